"""Speculative decoding over the block pool: the operators and a decoder that runs them.

A step takes, per sequence, a tree of drafted tokens behind the token emitted
last (node 0, the root, whose K/V is not cached yet) through ONE pass of the
model, and keeps the longest path that the target agrees with:

* ``tree_tables``     block tables, row starts, positions, slots and ancestor masks from request lengths, on the GPU;
* ``tree_attention``  every node over the cached positions and its own ancestors;
* ``target_probs``    logits to probabilities at a temperature per row;
* ``verify_tree``     accept / residual-resampling of the drafted tokens from given random numbers (or greedy);
* ``commit_tree``     the accepted path's K/V moved to consecutive positions in every layer.

``SpeculativeDecoder`` runs them with ``PromptLookup`` drafts (continuations
of earlier occurrences of the last tokens); its greedy stream is
``KshipraModel.generate``'s.  The reference's engine/speculative.py drafts and
verifies against a mock model only (speculative.py:51-81, 154-270).

All tensors are CUDA tensors on one device, which is checked; calls run on its
current stream and allocate only their outputs.  Errors that only the device can see are
OR-ed into ``flags`` (int32 [1], KSH_FLAG_* bits) where one is given.
"""

from __future__ import annotations

import functools
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib
from ._lib import ptr, stream_ptr

MAX_NODES = 256              # nodes of one sequence's tree: four 64-bit mask words


# These operators take 5 to 30 us on the GPU, so the host side of a call is kept
# short: the current stream's handle straight from torch (2 us less than through
# a Stream object), no device switch where the tensors' device is current.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _run(device: torch.device, name: str, *args) -> None:
    """The C entry on ``device`` and its current stream (appended to args)."""
    idx = device.index
    if idx != torch.cuda.current_device():
        with torch.cuda.device(device):
            _run(device, name, *args)
        return
    stream = _raw_stream(idx) if _raw_stream is not None else stream_ptr()
    st = getattr(_lib.lib(), name)(*args, stream)
    if st != 0:
        _lib.check(name, st)


def _wrong_device(name: str, at: int, dev: Optional[int]) -> Exception:
    if at < 0:
        return _lib.KshipraLibraryError(f"{name} must be a CUDA tensor (no CPU path)")
    return ValueError(f"{name} is on cuda:{at}, the call's other tensors on cuda:{dev}")


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, ndim: int,
          dev: Optional[int] = None) -> torch.Tensor:
    """``t`` if it fits and is on CUDA device ``dev`` (None: on any)."""
    at = t.get_device()
    if at < 0 or (at != dev and dev is not None):
        raise _wrong_device(name, at, dev)
    if t.dtype is not dtype or t.dim() != ndim or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {ndim}-D {dtype} tensor, got "
                         f"{t.dtype} {tuple(t.shape)}")
    return t


def _rows(t: torch.Tensor, name: str, dev: Optional[int] = None) -> torch.Tensor:
    """A 2-D fp32 tensor whose rows are contiguous (they may lie further apart)."""
    at = t.get_device()
    if at < 0 or (at != dev and dev is not None):
        raise _wrong_device(name, at, dev)
    if (t.dtype is not torch.float32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1)
            or (t.shape[0] > 1 and t.stride(0) < t.shape[1])):
        raise ValueError(f"{name} must be fp32 [rows, vocab] with contiguous rows, got "
                         f"{t.dtype} {tuple(t.shape)} strides {t.stride()}")
    return t


def _flags(t: Optional[torch.Tensor], dev: int) -> Optional[int]:
    """Address of the status word, or None."""
    if t is None:
        return None
    at = t.get_device()
    if at != dev:
        raise _wrong_device("flags", at, dev)
    if t.dtype is not torch.int32 or t.numel() < 1:
        raise ValueError(f"flags must be an int32 tensor of one element, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class TreeWorkspace:
    """Scratch of the tree attention, one buffer per device and stream (calls on
    different streams may overlap).  Needs no initialisation.

    A captured graph keeps the address that it was captured with, so a buffer is
    never replaced: it is allocated at the largest size of any head dimension
    (19.6 MB on 148 SMs).  And a call under capture gets a buffer of its own from
    the capture's memory pool, which lives as long as the graph: graphs captured
    on one stream may be replayed on several at once.
    """

    def __init__(self):
        self.bufs: Dict[tuple, torch.Tensor] = {}

    def get(self, nbytes: int, device: torch.device) -> torch.Tensor:
        idx = device.index
        if idx != torch.cuda.current_device():
            with torch.cuda.device(device):
                return self.get(nbytes, device)
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(nbytes, dtype=torch.uint8, device=device)
        key = (idx, _raw_stream(idx) if _raw_stream is not None else stream_ptr(device))
        buf = self.bufs.get(key)
        if buf is None:
            buf = self.bufs[key] = torch.empty(_largest_workspace(), dtype=torch.uint8, device=device)
        return buf


_WS = TreeWorkspace()


@functools.lru_cache(maxsize=None)
def _workspace_bytes(seqs: int, hq: int, hkv: int, d: int, max_nodes: int) -> int:
    return int(_lib.lib().ksh_tree_attention_workspace_size(seqs, hq, hkv, d, max_nodes))


@functools.lru_cache(maxsize=None)
def _largest_workspace() -> int:
    return max(_workspace_bytes(1, 1, 1, d, 1) for d in (64, 128))


def tree_tables(prefix_lens: torch.Tensor, new_lens: torch.Tensor, total: int, block_size: int,
                max_nodes: int, max_blocks: int, *, block_ids: Optional[torch.Tensor] = None,
                block_start: Optional[torch.Tensor] = None,
                block_tables: Optional[torch.Tensor] = None,
                parents: Optional[torch.Tensor] = None,
                flags: Optional[torch.Tensor] = None):
    """Tables of a batch from its request lengths.

    prefix_lens, new_lens int32 [S] (cached positions, rows of this pass);
    ``total`` the host's sum of new_lens; either block_ids int32 (every
    sequence's blocks in turn) with block_start int32 [S + 1], or ready
    block_tables int32 [S, max_blocks]; parents int32 [total] (own sequence's
    node index, negative for a root) or None for plain chunks.  Returns
    (q_start [S + 1], block_tables, positions [total], slots [total], mask
    [total, ceil(max_nodes / 64)] or None), as ``KshipraModel`` takes them.
    """
    S = prefix_lens.shape[0]
    at = _need(prefix_lens, "prefix_lens", torch.int32, 1).get_device()
    _need(new_lens, "new_lens", torch.int32, 1, at)
    if new_lens.shape[0] != S:
        raise ValueError("prefix_lens and new_lens differ in length")
    if (block_ids is None) != (block_start is None) or (block_ids is None) == (block_tables is None):
        raise ValueError("pass block_ids with block_start, or block_tables")
    dev = prefix_lens.device
    if block_ids is not None:
        _need(block_ids, "block_ids", torch.int32, 1, at)
        if _need(block_start, "block_start", torch.int32, 1, at).shape[0] != S + 1:
            raise ValueError("block_start must have one entry more than there are sequences")
        block_tables = prefix_lens.new_empty((S, max_blocks))
    elif tuple(_need(block_tables, "block_tables", torch.int32, 2, at).shape) != (S, max_blocks):
        raise ValueError(f"block_tables must be [{S}, {max_blocks}]")
    words = 0
    if parents is not None:
        if _need(parents, "parents", torch.int32, 1, at).shape[0] != total:
            raise ValueError("parents must have one entry per row")
        if not 1 <= max_nodes <= MAX_NODES:
            raise ValueError(f"max_nodes must be 1..{MAX_NODES}, got {max_nodes}")
        words = (max_nodes + 63) >> 6
    q_start = prefix_lens.new_empty(S + 1)
    positions = torch.empty(total, dtype=torch.int64, device=dev)
    slots = torch.empty_like(positions)
    mask = None if parents is None else positions.new_empty((total, words))
    _run(dev, "ksh_tree_tables", prefix_lens.data_ptr(), new_lens.data_ptr(), S, total, block_size,
         ptr(block_ids), 0 if block_ids is None else block_ids.shape[0], ptr(block_start),
         max_blocks, ptr(parents), words, q_start.data_ptr(), block_tables.data_ptr(),
         positions.data_ptr(), slots.data_ptr(), ptr(mask), _flags(flags, at))
    return q_start, block_tables, positions, slots, mask


def tree_attention(q: torch.Tensor, pool: torch.Tensor, layer: int, block_tables: torch.Tensor,
                   q_start: torch.Tensor, prefix_lens: torch.Tensor,
                   mask: Optional[torch.Tensor], max_nodes: int, max_total_len: int,
                   out: Optional[torch.Tensor] = None, flags: Optional[torch.Tensor] = None,
                   ws: TreeWorkspace = _WS) -> torch.Tensor:
    """Attention of drafted nodes over the pool: q [T, Hq, D] fp32 rotated
    queries, pool [nb, L, 2, Hkv, B, D] fp32 holding the nodes' own K/V in the
    slots of positions prefix .. prefix + n - 1, mask int64 [T, words] from
    ``tree_tables`` (None: node i attends nodes 0 .. i).  Returns [T, Hq, D];
    a node that may see no key gives zeros."""
    at = _need(q, "q", torch.float32, 3).get_device()
    _need(pool, "pool", torch.float32, 6, at)
    _need(block_tables, "block_tables", torch.int32, 2, at)
    T, hq, d = q.shape
    nb, L, two, hkv, bs, dp = pool.shape
    S, max_blocks = block_tables.shape
    if two != 2 or dp != d or hq % hkv != 0:
        raise ValueError(f"q {tuple(q.shape)} does not fit the pool {tuple(pool.shape)}")
    if not 0 <= layer < L:
        raise ValueError(f"layer {layer} outside the pool's {L}")
    if (_need(q_start, "q_start", torch.int32, 1, at).shape[0] != S + 1
            or _need(prefix_lens, "prefix_lens", torch.int32, 1, at).shape[0] != S):
        raise ValueError("q_start must have S + 1 and prefix_lens S entries")
    if not 0 <= max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes must be 0..{MAX_NODES}, got {max_nodes}")
    words = 0
    if mask is not None:
        if _need(mask, "mask", torch.int64, 2, at).shape[0] != T:
            raise ValueError("mask must have one row per node")
        words = mask.shape[1]
    if out is None:
        out = torch.empty_like(q)
    elif _need(out, "out", torch.float32, 3, at).shape != q.shape:
        raise ValueError("out must have q's shape")
    dev = q.device
    buf = ws.get(_workspace_bytes(S, hq, hkv, d, max_nodes), dev)
    _run(dev, "ksh_tree_attention", q.data_ptr(), T, hq, d, pool.data_ptr(), nb, L, layer, hkv, bs,
         block_tables.data_ptr(), max_blocks, q_start.data_ptr(), prefix_lens.data_ptr(), S,
         ptr(mask), words, max_nodes, max_total_len, out.data_ptr(), buf.data_ptr(), buf.numel(),
         _flags(flags, at))
    return out


def target_probs(logits: torch.Tensor, temperature: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Probabilities of logits [m, vocab] at temperature fp32 [m] (None: 1; 0:
    one at the first maximum).  ``out`` may be ``logits``."""
    m, vocab = _rows(logits, "logits").shape
    at = logits.get_device()
    if temperature is not None and _need(temperature, "temperature", torch.float32, 1, at).shape[0] != m:
        raise ValueError("temperature must have one entry per row")
    if out is None:
        out = torch.empty((m, vocab), dtype=torch.float32, device=logits.device)
    elif _rows(out, "out", at).shape != logits.shape:
        raise ValueError("out must have the logits' shape")
    _run(logits.device, "ksh_target_probs", logits.data_ptr(), m, vocab, _stride(logits),
         ptr(temperature), out.data_ptr(), _stride(out))
    return out


def verify_tree(tokens: torch.Tensor, parents: torch.Tensor, q_start: torch.Tensor,
                max_nodes: int, *, target_probs: Optional[torch.Tensor] = None,
                draft_probs: Optional[torch.Tensor] = None,
                target_tokens: Optional[torch.Tensor] = None,
                u_accept: Optional[torch.Tensor] = None, u_sample: Optional[torch.Tensor] = None,
                flags: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accepted path of each sequence's tree and the token after it.

    tokens int64 [T], parents int32 [T], q_start int32 [S + 1]; either
    target_probs fp32 [T, vocab] (the target's distribution after each node)
    with u_accept [T], u_sample [S] in [0, 1), and draft_probs [T, vocab] (the
    distribution a node's children were drawn from; None: fixed proposals), or
    target_tokens int64 [T] (greedy).  Returns (path int32 [S, max_nodes]
    padded with -1, path_len int32 [S], next int64 [S])."""
    T = _need(tokens, "tokens", torch.int64, 1).shape[0]
    at = tokens.get_device()
    S = _need(q_start, "q_start", torch.int32, 1, at).shape[0] - 1
    if _need(parents, "parents", torch.int32, 1, at).shape[0] != T or S < 1:
        raise ValueError("parents must have one entry per token, q_start S + 1 >= 2")
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError(f"max_nodes must be 1..{MAX_NODES}, got {max_nodes}")
    if (target_probs is None) == (target_tokens is None):
        raise ValueError("pass target_probs or target_tokens")
    vocab, ps, qs = 1 << 30, 0, 0
    if target_probs is not None:
        if u_accept is None or u_sample is None:
            raise ValueError("target_probs needs u_accept and u_sample")
        if _rows(target_probs, "target_probs", at).shape[0] != T:
            raise ValueError("target_probs must have one row per node")
        if (_need(u_accept, "u_accept", torch.float32, 1, at).shape[0] != T
                or _need(u_sample, "u_sample", torch.float32, 1, at).shape[0] != S):
            raise ValueError("u_accept must have one entry per node, u_sample per sequence")
        vocab, ps = target_probs.shape[1], _stride(target_probs)
        if draft_probs is not None:
            if _rows(draft_probs, "draft_probs", at).shape != target_probs.shape:
                raise ValueError("draft_probs must have target_probs' shape")
            qs = _stride(draft_probs)
    else:
        if draft_probs is not None:
            raise ValueError("draft_probs needs target_probs")
        if _need(target_tokens, "target_tokens", torch.int64, 1, at).shape[0] != T:
            raise ValueError("target_tokens must have one entry per node")
    dev = tokens.device
    path = q_start.new_empty((S, max_nodes))
    path_len = q_start.new_empty(S)
    nxt = tokens.new_empty(S)
    _run(dev, "ksh_verify_tree", tokens.data_ptr(), parents.data_ptr(), q_start.data_ptr(), S, T,
         max_nodes, vocab, ptr(target_probs), ps, ptr(draft_probs), qs, ptr(target_tokens),
         None if target_probs is None else u_accept.data_ptr(),
         None if target_probs is None else u_sample.data_ptr(), path.data_ptr(),
         path_len.data_ptr(), nxt.data_ptr(), _flags(flags, at))
    return path, path_len, nxt


def commit_tree(pool: torch.Tensor, block_tables: torch.Tensor, prefix_lens: torch.Tensor,
                path: torch.Tensor, path_len: torch.Tensor,
                flags: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Moves the K/V of each sequence's accepted nodes (path int32 [S, n],
    path_len int32 [S], from ``verify_tree``) to positions prefix, prefix + 1,
    ... in every layer of the pool, in place, and returns the new lengths
    prefix_lens + path_len (int32 [S])."""
    at = _need(pool, "pool", torch.float32, 6).get_device()
    nb, L, two, hkv, bs, d = pool.shape
    S, max_blocks = _need(block_tables, "block_tables", torch.int32, 2, at).shape
    if two != 2:
        raise ValueError(f"pool must be [nb, L, 2, Hkv, B, D], got {tuple(pool.shape)}")
    if (_need(prefix_lens, "prefix_lens", torch.int32, 1, at).shape[0] != S
            or _need(path_len, "path_len", torch.int32, 1, at).shape[0] != S
            or _need(path, "path", torch.int32, 2, at).shape[0] != S):
        raise ValueError("prefix_lens, path and path_len must have one entry per sequence")
    new_lens = prefix_lens.new_empty(S)
    _run(pool.device, "ksh_tree_commit", pool.data_ptr(), nb, L, hkv, bs, d,
         block_tables.data_ptr(), max_blocks, prefix_lens.data_ptr(), S, path.data_ptr(),
         path.shape[1], path_len.data_ptr(), new_lens.data_ptr(), _flags(flags, at))
    return new_lens


# ---------------------------------------------------------------------------
# drafts and the decode loop
# ---------------------------------------------------------------------------

class PromptLookup:
    """Drafts without a draft model: the continuations of up to ``branches``
    earlier occurrences of the last ``ngram`` (then fewer) tokens, latest
    first, merged into one tree of at most ``max_nodes`` nodes."""

    def __init__(self, ngram: int = 3, depth: int = 6, branches: int = 3, max_nodes: int = 16):
        if ngram < 1 or depth < 0 or branches < 0 or not 1 <= max_nodes <= MAX_NODES:
            raise ValueError("ngram >= 1, depth >= 0, branches >= 0, "
                             f"1 <= max_nodes <= {MAX_NODES}")
        self.ngram, self.depth, self.branches, self.max_nodes = ngram, depth, branches, max_nodes

    def propose(self, tokens: Sequence[int]) -> Tuple[List[int], List[int]]:
        """(node tokens, parents); node 0 is the last token.  Looks through all of
        ``tokens``; ``sequence`` is for one that grows."""
        n = len(tokens)

        def ends():
            for k in range(min(self.ngram, n - 1), 0, -1):
                tail = list(tokens[n - k:])
                for i in range(n - k - 1, -1, -1):
                    if list(tokens[i:i + k]) == tail:
                        yield i + k
        return self._tree(tokens, ends())

    def sequence(self, tokens: Sequence[int]):
        """A growing sequence: ``extend(tokens)`` and ``propose()``."""
        return _LookupSequence(self, tokens)

    def _tree(self, tokens: Sequence[int], ends) -> Tuple[List[int], List[int]]:
        """The tree of the continuations from ``ends``, the places behind earlier
        occurrences of the last tokens, in order."""
        out, parents = [int(tokens[-1])], [-1]
        children: Dict[Tuple[int, int], int] = {}
        seen = set()
        if self.branches < 1 or self.max_nodes < 2:
            return out, parents
        for end in ends:
            if end in seen:
                continue
            seen.add(end)
            at = 0
            for t in tokens[end:end + self.depth]:
                nxt = children.get((at, int(t)))
                if nxt is None:
                    if len(out) >= self.max_nodes:
                        break
                    nxt = len(out)
                    out.append(int(t))
                    parents.append(at)
                    children[(at, int(t))] = nxt
                at = nxt
            if len(seen) >= self.branches or len(out) >= self.max_nodes:
                break
        return out, parents


class _LookupSequence:
    """``PromptLookup`` on one growing sequence.  For each length k an n-gram's
    latest end, and for each end the one before it: a proposal follows at most
    ``branches`` links and a new token adds one per length.  On one core of the
    host 1 to 6 us a proposal and 1.3 us a token at any length, after 6 ms for a
    prompt of 4096; looking through the history takes 2 ms at 4096 tokens and 20
    at 31000 where nothing matches, for every step."""

    def __init__(self, lookup: PromptLookup, tokens: Sequence[int]):
        self.lookup = lookup
        self.tokens: List[int] = []
        self.latest = [{} for _ in range(lookup.ngram)]             # k - 1: n-gram -> end
        self.before: List[List[int]] = [[] for _ in range(lookup.ngram)]   # k - 1: [end - k] -> end, 0: none
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            self.tokens.append(int(t))
            end = len(self.tokens)
            for k in range(1, min(self.lookup.ngram, end) + 1):
                gram = tuple(self.tokens[end - k:end])
                self.before[k - 1].append(self.latest[k - 1].get(gram, 0))
                self.latest[k - 1][gram] = end

    def propose(self) -> Tuple[List[int], List[int]]:
        n = len(self.tokens)

        def ends():
            for k in range(min(self.lookup.ngram, n - 1), 0, -1):
                end = self.before[k - 1][n - k]
                while end:
                    yield end
                    end = self.before[k - 1][end - k]
        return self.lookup._tree(self.tokens, ends())


class _WholeSequence:
    """A growing sequence for a proposer that takes all of its tokens each time."""

    def __init__(self, proposer, tokens: Sequence[int]):
        self.proposer, self.tokens = proposer, list(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        self.tokens.extend(tokens)

    def propose(self) -> Tuple[List[int], List[int]]:
        return self.proposer.propose(list(self.tokens))


def sequence_of(proposer, tokens: Sequence[int]):
    """``proposer.sequence(tokens)`` where it has one that goes with its ``propose``."""
    kind = type(proposer)
    own = getattr(kind, "sequence", None)
    if own is None or (own is PromptLookup.sequence and kind.propose is not PromptLookup.propose):
        return _WholeSequence(proposer, tokens)
    return proposer.sequence(tokens)


def cut_tree(tokens: Sequence[int], parents: Sequence[int], depth: int
             ) -> Tuple[List[int], List[int]]:
    """The nodes at most ``depth`` below their root, renumbered.  A parent that
    is no earlier node becomes -1 (which the verification reports)."""
    if len(tokens) < 1 or len(tokens) != len(parents):
        raise ValueError(f"a tree needs a token and a parent per node, got {len(tokens)} and {len(parents)}")
    if depth >= len(tokens) - 1:                 # a chain of all of them is no deeper
        return list(tokens), list(parents)
    below: List[int] = []
    at: List[int] = []
    toks, ups = [], []
    for i, (t, p) in enumerate(zip(tokens, parents)):
        inner = 0 <= p < i
        below.append(below[p] + 1 if inner else 0)
        at.append(len(toks))
        if below[i] <= depth:
            toks.append(t)
            ups.append(at[p] if inner else -1)
    return toks, ups


class SpeculativeDecoder:
    """Batched decoding of drafted trees through a ``KshipraModel``.

    ``generate(prompts, max_new_tokens)`` prefills each prompt and then runs
    one verified tree per sequence and step.  temperature 0 is greedy (the
    tokens of ``KshipraModel.generate``); above, tokens follow the target's
    distribution at that temperature, with random numbers from ``generator``.
    ``proposer`` has ``max_nodes`` and ``propose(tokens) -> (tokens, parents)``, or
    ``sequence(tokens)`` for an object with ``extend(tokens)`` and ``propose()``.
    After a run, ``steps`` and ``emitted`` hold the passes and tokens counted.
    """

    def __init__(self, model, proposer=None, block_size: int = 16, temperature: float = 0.0,
                 generator: Optional[torch.Generator] = None):
        if temperature > 0 and model.tp_world > 1:
            raise ValueError("sampling needs the whole vocabulary on one GPU")
        if getattr(model, "kv_dtype", torch.float32) != torch.float32:
            raise ValueError("drafted trees need an fp32 pool (kv_dtype)")
        self.m = model
        self.proposer = proposer if proposer is not None else PromptLookup()
        self.block_size = block_size
        self.temperature = float(temperature)
        self.generator = generator
        self.steps = 0
        self.emitted = 0
        self._ws = TreeWorkspace()

    @torch.inference_mode()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 20,
                 eos_token_id: Optional[int] = None,
                 prefill_chunk: Optional[int] = None) -> List[List[int]]:
        from .model import _check_flags
        m, bs = self.m, self.block_size
        if max_new_tokens < 1 or any(len(p) < 1 for p in prompts):
            raise ValueError("prompts need a token and max_new_tokens must be positive")
        self.steps = self.emitted = 0
        with torch.cuda.device(m.device):
            spare = self.proposer.max_nodes
            need = [(len(p) + max_new_tokens + spare + bs - 1) // bs for p in prompts]
            pool = m.new_pool(sum(need), bs).pool
            at, tables = 0, []
            for n in need:
                tables.append(list(range(at, at + n)))
                at += n
            out: List[List[int]] = []
            for p, bt in zip(prompts, tables):
                out.append([self._first(p, pool, bt, prefill_chunk)])
            _check_flags(m.flags)
            self.emitted = len(out)
            live = [i for i in range(len(out)) if not self._done(out[i], max_new_tokens, eos_token_id)]
            seqs = {i: sequence_of(self.proposer, list(prompts[i]) + out[i]) for i in live}
            while live:
                self._step(prompts, seqs, out, tables, pool, live, max_new_tokens, eos_token_id)
                live = [i for i in live if not self._done(out[i], max_new_tokens, eos_token_id)]
        return out

    @staticmethod
    def _done(toks: List[int], most: int, eos: Optional[int]) -> bool:
        return len(toks) >= most or (eos is not None and toks[-1] == eos)

    def _rand(self, n: int) -> torch.Tensor:
        return torch.rand(n, generator=self.generator, device=self.m.device)

    def _first(self, prompt, pool, bt, chunk) -> int:
        m = self.m
        if self.temperature <= 0:
            return int(m.prefill(prompt, pool, bt, chunk).item())
        # the prompt's last token is the root of a tree of one node
        if len(prompt) > 1:
            m.prefill(prompt[:-1], pool, bt, chunk)
        _, _, nxt = self._pass(pool, [bt], [len(prompt) - 1], [[int(prompt[-1])]], [[-1]])
        return int(nxt.item())

    def _pass(self, pool, tables, prefix, toks, parents):
        """One pass of the model over the trees; (path, path_len, next), committed."""
        from .model import _check_flags
        m, dev, bs = self.m, self.m.device, self.block_size
        S, lens = len(toks), [len(t) for t in toks]
        T, most = sum(lens), max(lens)
        blocks = [(p + n + bs - 1) // bs for p, n in zip(prefix, lens)]
        start = [0]
        for b in blocks:
            start.append(start[-1] + b)
        # one host-to-device copy: lengths, blocks, tokens and parents
        flat = (prefix + lens + start + [b for bt, n in zip(tables, blocks) for b in bt[:n]]
                + [t for x in toks for t in x] + [p for x in parents for p in x])
        buf = torch.tensor(flat, dtype=torch.int32).to(dev)
        pre, new, bst, ids, tok32, par = buf.split([S, S, S + 1, start[-1], T, T])
        tok = tok32.long()
        q_start, bt, pos, slots, mask = tree_tables(pre, new, T, bs, most, max(blocks),
                                                    block_ids=ids, block_start=bst, parents=par,
                                                    flags=m.flags)
        max_total = max(p + n for p, n in zip(prefix, lens))
        acts = m._alloc_acts(T)
        hid = m._run_layers(acts, tok, pos, slots, bt, q_start, pre, S, most, max_total, pool,
                            m._lin_ws, m._attn_ws, tree=(mask, self._ws))
        best = torch.empty(T, dtype=torch.int64, device=dev)
        if self.temperature <= 0:
            m._lm_head_argmax(hid, best)
            path, path_len, nxt = verify_tree(tok, par, q_start, most, target_tokens=best,
                                              flags=m.flags)
        else:
            logits = torch.empty((T, m.vocab_size), dtype=torch.float32, device=dev)
            m._lm_head_argmax(hid, best, logits=logits)
            temp = torch.full((T,), self.temperature, device=dev)
            probs = target_probs(logits, temp, out=logits)
            path, path_len, nxt = verify_tree(tok, par, q_start, most, target_probs=probs,
                                              u_accept=self._rand(T), u_sample=self._rand(S),
                                              flags=m.flags)
        commit_tree(pool, bt, pre, path, path_len, flags=m.flags)
        _check_flags(m.flags)
        return path, path_len, nxt

    def _step(self, prompts, seqs, out, tables, pool, live, most: int, eos: Optional[int]) -> None:
        prefix, toks, parents = [], [], []
        for i in live:
            have = len(prompts[i]) + len(out[i])
            t, p = seqs[i].propose()
            if len(t) > self.proposer.max_nodes:
                raise ValueError(f"{len(t)} drafted nodes, max_nodes is {self.proposer.max_nodes}")
            # a step emits one token more than it accepts; nothing past the
            # position table can be accepted
            t, p = cut_tree(t, p, max(0, min(most - len(out[i]) - 1, self.m.max_positions - have)))
            prefix.append(have - 1)
            toks.append(t)
            parents.append(p)
        path, path_len, nxt = self._pass(pool, [tables[i] for i in live], prefix, toks, parents)
        for i, t, row, n, last in zip(live, toks, path.tolist(), path_len.tolist(), nxt.tolist()):
            new = [t[j] for j in row[1:n]] + [last]
            new = new[:most - len(out[i])]
            if eos is not None and eos in new:
                new = new[:new.index(eos) + 1]
            out[i].extend(new)
            seqs[i].extend(new)
            self.emitted += len(new)
        self.steps += 1
