"""A 16-bit paged K/V cache: the pass that writes it, the attention that reads
it, and the operations on its pages.

The pool is the ``BlockAllocator``'s (``[num_blocks, num_layers, 2, Hkv, B,
D]``) in fp16 or bf16: half of the bytes of an fp32 pool, for the cache and for
every decode step that reads it.  Queries, outputs and everything that is summed
stay fp32; K and V are rounded once, when they are stored.

* ``rope_cache_write``  norms of queries and keys per head (where a model has them), position rotation, K/V into the pool;
* ``cache_attention``   a chunk of new tokens of each sequence (one while decoding) over its cached positions;
* ``fork_pages``        sequences continued by others (beams): whole pages shared, the page being filled copied;
* ``compact_pages``     the pages in use moved to the front of the pool.

``KshipraModel(kv_dtype=...)`` runs the first two, ``BeamDecoder`` the third,
``PrefixCache.compact`` the fourth.

All tensors are CUDA tensors on one device, which is checked; calls run on its
current stream and allocate only their outputs and scratch.  Errors that only the
device can see are OR-ed into ``flags`` (int32 [1], KSH_FLAG_* bits) where one is
given.
"""

from __future__ import annotations

import functools
import threading
from typing import Dict, Optional, Tuple

import torch

from . import _lib
from ._lib import ptr, stream_ptr
from .speculative import _flags, _need, _raw_stream, _run, _wrong_device

POOL_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_SEQS = 65535             # sequences of one call of ksh_cache_attention's general kernel


def _pool(t: torch.Tensor, types, dev: Optional[int] = None) -> int:
    """The KSH_TYPE_* of a pool on device ``dev`` (None: any)."""
    at = t.get_device()
    if at < 0 or (at != dev and dev is not None):
        raise _wrong_device("pool", at, dev)
    kind = POOL_TYPES.get(t.dtype, -1)
    if kind not in types or t.dim() != 6 or t.shape[2] != 2 or not t.is_contiguous():
        names = ", ".join(str(k)[6:] for k, v in POOL_TYPES.items() if v in types)
        raise ValueError(f"pool must be a contiguous [nb, L, 2, Hkv, B, D] tensor of {names}, got "
                         f"{t.dtype} {tuple(t.shape)}")
    return kind


class CacheWorkspace:
    """Scratch of the cache attention, one buffer per device and stream (calls on
    different streams may overlap), of the largest size of any head dimension, so that
    it is never replaced under a captured graph.  Needs no initialisation.  A call
    under capture gets a buffer of its own from the capture's memory pool, which
    lives as long as the graph: graphs captured on one stream may be replayed on
    several at once."""

    def __init__(self):
        self.bufs: Dict[tuple, torch.Tensor] = {}
        self.lock = threading.Lock()          # held over a call's launches: threads may share a stream

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


_WS = CacheWorkspace()


@functools.lru_cache(maxsize=None)
def _workspace_bytes(d: int) -> int:
    """Of any call with this head dimension: the size depends on nothing else."""
    return int(_lib.lib().ksh_cache_attention_workspace_size(1, 1, 1, d, 1))


@functools.lru_cache(maxsize=None)
def _largest_workspace() -> int:
    return max(_workspace_bytes(d) for d in (64, 128))


def rope_cache_write(qkv: torch.Tensor, pool: torch.Tensor, layer: int, positions: torch.Tensor,
                     slots: torch.Tensor, rope_cos: torch.Tensor, rope_sin: torch.Tensor, *,
                     q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                     eps: float = 1e-6, out: Optional[torch.Tensor] = None,
                     flags: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of q, k and v (qkv fp32 [T, (Hq + 2 Hkv) D]) into the cache.

    q and k heads are normed where a weight fp32 [D] is given (w * x /
    sqrt(mean(x^2) + eps)) and rotated at positions int64 [T] by the tables fp32
    [max_pos, D / 2]; k and v go, rounded to the pool's type (fp32, fp16, bf16), into
    slots int64 [T] (block * B + offset, distinct) of ``layer``.  Returns the
    queries fp32 [T, Hq, D]."""
    at = _need(qkv, "qkv", torch.float32, 2).get_device()
    kind = _pool(pool, (0, 1, 2), at)
    nb, L, _, hkv, bs, d = pool.shape
    T, width = qkv.shape
    hq = width // d - 2 * hkv
    if width % d or hq < 1 or d % 2:
        raise ValueError(f"qkv {tuple(qkv.shape)} does not fit the pool {tuple(pool.shape)}")
    if not 0 <= layer < L:
        raise ValueError(f"layer {layer} outside the pool's {L}")
    if (_need(positions, "positions", torch.int64, 1, at).shape[0] != T
            or _need(slots, "slots", torch.int64, 1, at).shape[0] != T):
        raise ValueError("positions and slots must have one entry per row")
    if (_need(rope_cos, "rope_cos", torch.float32, 2, at).shape[1] * 2 != d
            or _need(rope_sin, "rope_sin", torch.float32, 2, at).shape != rope_cos.shape):
        raise ValueError(f"rope_cos and rope_sin must be [max_pos, {d // 2}]")
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None and _need(w, name, torch.float32, 1, at).shape[0] != d:
            raise ValueError(f"{name} must have {d} entries")
    if out is None:
        out = torch.empty((T, hq, d), dtype=torch.float32, device=qkv.device)
    elif tuple(_need(out, "out", torch.float32, 3, at).shape) != (T, hq, d):
        raise ValueError(f"out must be [{T}, {hq}, {d}]")
    _run(qkv.device, "ksh_rope_cache_write", qkv.data_ptr(), T, hq, hkv, d, positions.data_ptr(),
         slots.data_ptr(), rope_cos.data_ptr(), rope_sin.data_ptr(), rope_cos.shape[0], ptr(q_norm),
         ptr(k_norm), eps, out.data_ptr(), pool.data_ptr(), kind, nb, L, layer, bs, _flags(flags, at))
    return out


def cache_attention(q: torch.Tensor, pool: torch.Tensor, layer: int, block_tables: torch.Tensor,
                    q_start: torch.Tensor, prefix_lens: torch.Tensor, max_q_len: int,
                    max_total_len: int, out: Optional[torch.Tensor] = None,
                    flags: Optional[torch.Tensor] = None,
                    ws: CacheWorkspace = _WS) -> torch.Tensor:
    """Attention of new tokens over a 16-bit pool.

    q fp32 [T, Hq, D] rotated queries; pool [nb, L, 2, Hkv, B, D] fp16 or bf16,
    holding the new tokens' own K/V too; block_tables int32 [S, max_blocks]; rows
    q_start[s] .. q_start[s + 1] - 1 (int32 [S + 1]) are sequence s's, at positions
    prefix_lens[s] (int32 [S]) and on, and attend every position up to their own.
    ``max_q_len`` bounds a sequence's rows, ``max_total_len`` (its positions) only
    sizes the launch.
    Returns fp32 [T, Hq, D]; rows of q that no sequence covers are not written."""
    at = _need(q, "q", torch.float32, 3).get_device()
    kind = _pool(pool, (1, 2), at)
    _need(block_tables, "block_tables", torch.int32, 2, at)
    T, hq, d = q.shape
    nb, L, _, hkv, bs, dp = pool.shape
    S, max_blocks = block_tables.shape
    if dp != d or hq % hkv != 0:
        raise ValueError(f"q {tuple(q.shape)} does not fit the pool {tuple(pool.shape)}")
    if not 0 <= layer < L:
        raise ValueError(f"layer {layer} outside the pool's {L}")
    if (_need(q_start, "q_start", torch.int32, 1, at).shape[0] != S + 1
            or _need(prefix_lens, "prefix_lens", torch.int32, 1, at).shape[0] != S):
        raise ValueError("q_start must have S + 1 and prefix_lens S entries")
    if max_q_len < 0 or max_total_len < 0:
        raise ValueError("max_q_len and max_total_len must not be negative")
    if out is None:
        out = torch.empty_like(q)
    elif _need(out, "out", torch.float32, 3, at).shape != q.shape:
        raise ValueError("out must have q's shape")
    dev = q.device
    step = S
    if S > MAX_SEQS and not (d in (64, 128) and hq // hkv <= 128 and pool.numel() // d < 1 << 31
                             and (q.data_ptr() | pool.data_ptr() | out.data_ptr()) % 16 == 0):
        step = MAX_SEQS                      # a call of the general kernel: runs of sequences
    with ws.lock:
        buf = ws.get(_workspace_bytes(d), dev)
        for s in range(0, max(S, 1), max(step, 1)):
            _run(dev, "ksh_cache_attention", q.data_ptr(), T, hq, d, pool.data_ptr(), kind, nb, L, layer,
                 hkv, bs, block_tables.data_ptr() + 4 * s * max_blocks, max_blocks, q_start.data_ptr() + 4 * s,
                 prefix_lens.data_ptr() + 4 * s, min(step, S - s), max_q_len, max_total_len, out.data_ptr(),
                 buf.data_ptr(), buf.numel(), _flags(flags, at))
    return out


def fork_pages(pool: torch.Tensor, block_tables: torch.Tensor, lens: torch.Tensor,
               parents: torch.Tensor, ref_counts: torch.Tensor,
               flags: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Sequences continued by others.

    block_tables int32 [S, max_blocks] and lens int32 [S] (tokens cached) describe
    the old sequences, parents int32 [N] which of them each new one continues
    (negative: none), ref_counts int32 [nb] how many rows of all tables hold each
    page.  Whole pages are shared; the page that the next token goes to stays with
    the first child that continues in it, where no row but the old ones holds it,
    and is copied for the others (its filled rows, in every layer of the pool, in
    place), and where a page begins each child gets a free one: the lowest pages whose count is 0 once the old sequences gave up
    theirs.  With parents 0 .. S - 1 the call only grows the sequences, with
    negative ones it frees them.  Returns (block_tables [N, max_blocks], lens [N],
    slots int64 [N] of the next tokens, ref_counts [nb]); without a page left a slot is
    -1 and KSH_FLAG_NO_PAGE (512) raised.  A row whose slot is -1 takes no token and
    holds its whole pages alone: pass lens // B * B of it to the next call, which gives
    up the pages that its lens name."""
    kind = _pool(pool, (0, 1, 2))
    at = pool.get_device()
    nb, L, _, hkv, bs, d = pool.shape
    S, max_blocks = _need(block_tables, "block_tables", torch.int32, 2, at).shape
    N = _need(parents, "parents", torch.int32, 1, at).shape[0]
    if (_need(lens, "lens", torch.int32, 1, at).shape[0] != S
            or _need(ref_counts, "ref_counts", torch.int32, 1, at).shape[0] != nb):
        raise ValueError("lens must have one entry per sequence, ref_counts one per page")
    if max_blocks < 1:
        raise ValueError("block_tables need a column")
    # one allocation for the int32 outputs and the scratch (a tensor of its own takes
    # twice a view's time, and the host's time is most of a small call's)
    at_lens = N * max_blocks
    at_refs = at_lens + N
    scratch = S + 3 * N + 1
    buf = lens.new_empty(at_refs + nb + scratch)
    tables = buf.as_strided((N, max_blocks), (max_blocks, 1))
    new_lens = buf.as_strided((N,), (1,), at_lens)
    refs = buf.as_strided((nb,), (1,), at_refs)
    slots = torch.empty_like(parents, dtype=torch.int64)
    base = buf.data_ptr()
    _run(pool.device, "ksh_fork_pages", pool.data_ptr(), kind, nb, L, hkv, bs, d,
         block_tables.data_ptr(), max_blocks, lens.data_ptr(), S, parents.data_ptr(), N,
         ref_counts.data_ptr(), base, base + 4 * at_lens, slots.data_ptr(), base + 4 * at_refs,
         base + 4 * (at_refs + nb), scratch, _flags(flags, at))
    return tables, new_lens, slots, refs


def compact_pages(pool: torch.Tensor, block_tables: torch.Tensor, ref_counts: torch.Tensor
                  ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The u pages in use (ref_counts int32 [nb] above 0) moved to pages 0 .. u - 1.

    The k-th used page from u on goes to the k-th free page below u, in every
    layer, in place; the others stay.  Returns (block_tables renumbered, ref_counts
    at the new numbers, page_map int32 [nb] old -> new, u int32 [1])."""
    kind = _pool(pool, (0, 1, 2))
    at = pool.get_device()
    nb, L, _, hkv, bs, d = pool.shape
    _need(block_tables, "block_tables", torch.int32, 2, at)
    if _need(ref_counts, "ref_counts", torch.int32, 1, at).shape[0] != nb:
        raise ValueError("ref_counts must have one entry per page")
    rows, cols = block_tables.shape
    n = rows * cols
    buf = ref_counts.new_empty(n + 3 * nb + 3)             # one allocation, as in fork_pages
    tables = buf.as_strided((rows, cols), (cols, 1))
    refs = buf.as_strided((nb,), (1,), n)
    page_map = buf.as_strided((nb,), (1,), n + nb)
    used = buf.as_strided((1,), (1,), n + 2 * nb)
    base = buf.data_ptr()
    _run(pool.device, "ksh_compact_pages", pool.data_ptr(), kind, nb, L, hkv, bs, d,
         block_tables.data_ptr(), n, ref_counts.data_ptr(), base, base + 4 * n, base + 4 * (n + nb),
         base + 4 * (n + 2 * nb), base + 4 * (n + 2 * nb + 1), nb + 2)
    return tables, refs, page_map, used
