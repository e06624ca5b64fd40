"""Cases and plain forms of the operators of a 16-bit paged K/V cache.

Four operators that serving over such a cache runs next to each other:

* ``write``      a pass's q / k / v rows: norms of queries and keys for each head, position rotation, keys and values
                 rounded into their slots of the pool;
* ``attention``  a chunk of new tokens of each sequence (one token while decoding) over its cached positions;
* ``fork``       sequences continued by others (beams): whole pages shared, the page being filled copied, pages that
                 nobody holds any more freed, a fresh page where one begins;
* ``compact``    the pages in use moved to the front of the pool.

``run`` computes them in plain torch where ``own`` is false and through ``kshipra_b200.kv_cache`` where it is true.
``exact`` restates each from its definition in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #

def _attn(name, seqs, heads, kv_heads, head_dim, block, ctx, new, ragged, dtype, layers=1):
    return dict(name=name, op="attention", seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block=block, ctx=ctx,
                new=new, ragged=ragged, dtype=dtype, layers=layers)


def listed():
    return [
        # one interactive request of the 0.5B shape (14 / 2 heads of 64) decoding behind a 512-token prompt
        _attn("attn-1x540-one-h14", 1, 14, 2, 64, 16, 540, 1, False, "float16", layers=2),
        # the 8B shape's decode batch: 64 requests at context 4096, one token each
        _attn("attn-64x4096-one-h32", 64, 32, 8, 128, 16, 4096, 1, False, "float16"),
        # continuous batching of the 0.5B shape: 24 requests, prefill chunks among single tokens, an odd block size
        _attn("attn-24x2000-chunk301-h14", 24, 14, 2, 64, 24, 2000, 301, True, "bfloat16"),
        # the 8B shape's prefill chunk: 2048 tokens behind 4096 cached ones
        _attn("attn-1x4096-chunk2048-h32", 1, 32, 8, 128, 16, 4096, 2048, False, "float16"),
        # few long requests of the 8B heads, a chunk each
        _attn("attn-3x31000-chunk200-h32", 3, 32, 8, 128, 64, 31000, 200, True, "bfloat16"),
        # one token of the 0.5B shape
        dict(name="write-1-h14", op="write", rows=1, heads=14, kv_heads=2, head_dim=64, block=16, norm=False, dtype="float16"),
        # a prefill chunk of the 8B shape, in a model with norms of queries and keys
        dict(name="write-2048-h32-norm", op="write", rows=2048, heads=32, kv_heads=8, head_dim=128, block=16, norm=True,
             dtype="bfloat16"),
        # one request with four beams, 0.5B shape: 24 layers
        dict(name="fork-1x4-24xh2x64", op="fork", seqs=1, beams=4, layers=24, kv_heads=2, head_dim=64, block=16, ctx=540,
             dtype="float16"),
        # 16 requests with four beams each, 8B shape: 32 layers
        dict(name="fork-16x4-32xh8x128", op="fork", seqs=16, beams=4, layers=32, kv_heads=8, head_dim=128, block=16, ctx=75,
             dtype="float16"),
        # a small pool of the 0.5B shape after some requests left
        dict(name="compact-60-24xh2x64", op="compact", pages=60, used=31, seqs=3, layers=24, kv_heads=2, head_dim=64, block=16,
             dtype="float16"),
        # a pool of the 8B shape, half empty
        dict(name="compact-400-32xh8x128", op="compact", pages=400, used=210, seqs=20, layers=32, kv_heads=8, head_dim=128, block=16,
             dtype="bfloat16"),
    ]


HEADS = [(14, 2, 64), (32, 8, 128), (4, 2, 64), (16, 4, 128), (8, 2, 128), (8, 8, 64), (16, 2, 128)]
TYPES = ["float16", "bfloat16"]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["attention", "attention", "attention", "write", "fork", "compact"])
    h, hk, d = rng.choice(HEADS)
    c = dict(op=op, kv_heads=hk, head_dim=d, block=rng.choice([16, 24, 64, 10]), dtype=rng.choice(TYPES))
    if op == "attention":
        new = rng.choice([1, _log(rng, 1, 2048)])
        return dict(c, seqs=_log(rng, 1, 64), heads=h, ctx=_log(rng, 20, 31000), new=new, ragged=rng.random() < 0.7,
                    layers=rng.choice([1, 2]))
    if op == "write":
        return dict(c, rows=_log(rng, 1, 2048), heads=h, norm=rng.random() < 0.5)
    layers = rng.choice([2, 24, 32])
    if op == "fork":
        return dict(c, seqs=_log(rng, 1, 16), beams=rng.randint(1, 8), layers=layers, ctx=_log(rng, 1, 600))
    pages = _log(rng, 8, 400)
    return dict(c, pages=pages, used=rng.randint(1, pages), seqs=rng.randint(1, 20), layers=layers)


def _size(case):
    """What a pass and its preparation touch, in bytes, for the bound on drawn cases."""
    op = case["op"]
    if op == "attention":
        keys = case["ctx"] + case["new"]
        kv = 12.0 * case["seqs"] * keys * case["kv_heads"] * case["head_dim"] * case["layers"]
        return max(kv, 4.0 * case["seqs"] * keys * case["heads"] * case["new"])
    if op == "write":
        return work(case)["bytes"]
    page = 4.0 * case["layers"] * case["kv_heads"] * case["head_dim"] * case["block"]
    if op == "fork":
        return page * (case["seqs"] * (case["ctx"] // case["block"] + 2.0 * case["beams"] + 2) + 8)
    return 2.0 * page * case["pages"]


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _size(c))
    while True:
        c = _draw(rng)
        if _size(c) <= most[c["op"]]:
            return c


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #

def _lens(case):
    """Cached positions and new tokens of each sequence, from the case alone."""
    s, n, ctx = case["seqs"], case["new"], case["ctx"]
    if not case["ragged"]:
        return np.full(s, ctx, np.int64), np.full(s, n, np.int64)
    r = np.random.RandomState((s * 7919 + ctx * 31 + n * 17) % (1 << 31))
    pre = r.randint(ctx // 3, ctx + 1, s)
    new = r.randint((n + 1) // 2, n + 1, s)
    new[r.rand(s) < 0.5] = 1                              # half of the requests decode
    pre[r.rand(s) < 0.2] = 0                              # some begin
    pre[0], new[0] = ctx, n
    return pre.astype(np.int64), new.astype(np.int64)


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device=DEV, dtype=dtype)


def _fill(shape, dtype, g):
    """A pool of normal numbers, made in pieces (a generator fills 32 bits at a time)."""
    out = torch.empty(shape, dtype=getattr(torch, dtype), device=DEV)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 26):
        b = min(flat.numel(), a + (1 << 26))
        flat[a:b] = torch.randn(b - a, generator=g, device=DEV)
    return out


def _beams(case, rs):
    """Tables, lengths (from the case alone) and parents of requests whose beams share their pages but the last one."""
    s, k, b = case["seqs"], case["beams"], case["block"]
    r = np.random.RandomState((s * 7919 + case["ctx"] * 31 + k * 17) % (1 << 31))
    lens = np.repeat(r.randint((case["ctx"] + 1) // 2, case["ctx"] + 1, s), k)
    held = -(-lens // b)
    m = int(lens.max()) // b + 2
    total = int((lens[::k] // b).sum() + (lens % b > 0).sum())
    nb = total + s * k + 5                                # a fresh page for each child, and some
    ids = rs.permutation(nb)
    tables, refs, at = np.zeros((s * k, m), np.int64), np.zeros(nb, np.int64), 0
    for i in range(s):
        full = int(lens[i * k]) // b
        share = ids[at: at + full]
        at += full
        for j in range(i * k, i * k + k):
            tables[j, :full] = share
            if held[j] > full:
                tables[j, full] = ids[at]
                at += 1
    np.add.at(refs, np.concatenate([tables[j, : held[j]] for j in range(s * k)]), 1)
    # the best continuations come from a few of a request's beams; some requests have ended
    parents = (np.arange(s)[:, None] * k + np.minimum(rs.geometric(0.5, (s, k)) - 1, k - 1)).reshape(-1)
    parents[np.repeat(rs.rand(s) < 0.1, k)] = -1
    return tables, lens, parents, refs, nb


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    op, b, hk, d = case["op"], case["block"], case["kv_heads"], case["head_dim"]
    st = {"case": case}
    if op == "write":
        t = case["rows"]
        nb = -(-t // b) + 7
        st["qkv"] = randn(t, (case["heads"] + 2 * hk) * d) * 1.5
        st["positions"] = _dev(rs.randint(0, 4096) + np.arange(t), torch.int64)
        st["slots"] = _dev(rs.permutation(nb)[np.arange(t) // b] * b + np.arange(t) % b, torch.int64)
        inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, dtype=torch.float64) / d))
        ang = torch.outer(torch.arange(8192, dtype=torch.float64), inv)
        st["cos"], st["sin"] = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
        st["q_norm"] = 1.0 + 0.1 * randn(d) if case["norm"] else None
        st["k_norm"] = 1.0 + 0.1 * randn(d) if case["norm"] else None
        st["pool"] = torch.zeros(nb, 1, 2, hk, b, d, dtype=getattr(torch, case["dtype"]), device=DEV)
        st["out"] = torch.empty(t, case["heads"], d, device=DEV)
        return st
    if op == "attention":
        pre, new = _lens(case)
        need = -(-(pre + new) // b)
        start = np.concatenate([[0], np.cumsum(need)])
        nb = int(start[-1]) + 3
        ids = rs.permutation(nb)
        table = np.zeros((case["seqs"], int(need.max())), np.int64)
        for i in range(case["seqs"]):
            table[i, : need[i]] = ids[start[i]: start[i + 1]]
        qs = np.concatenate([[0], np.cumsum(new)])
        st.update(block_tables=_dev(table, torch.int32), q_start=_dev(qs, torch.int32), prefix_lens=_dev(pre, torch.int32),
                  total=int(qs[-1]), max_new=int(new.max()), max_total=int((pre + new).max()), layer=case["layers"] - 1)
        st["pool"] = _fill((nb, case["layers"], 2, hk, b, d), case["dtype"], g)
        # after the rotation queries are larger than keys in trained models: scores spread over several units
        st["q"] = randn(st["total"], case["heads"], d) * 2.0
        st["out"] = torch.empty_like(st["q"])
        return st
    if op == "fork":
        tables, lens, parents, refs, nb = _beams(case, rs)
        st["lens"], st["parents"] = _dev(lens, torch.int32), _dev(parents, torch.int32)
    else:
        nb, u = case["pages"], case["used"]
        used = rs.permutation(nb)[:u]
        refs = np.zeros(nb, np.int64)
        refs[used] = rs.randint(1, 4, u)
        tables = rs.choice(used, (case["seqs"], max(1, u // case["seqs"])))
    st["block_tables"], st["ref_counts"] = _dev(tables, torch.int32), _dev(refs, torch.int32)
    st["pool"] = _fill((nb, case["layers"], 2, hk, b, d), case["dtype"], g)
    return st


# --------------------------------------------------------------------------- #
# plain forms
# --------------------------------------------------------------------------- #

def _plain_write(st):
    case = st["case"]
    h, hk, d, b = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    q, k, v = st["qkv"].view(-1, h + 2 * hk, d).split([h, hk, hk], 1)

    def turn(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        c, s = st["cos"][st["positions"]][:, None], st["sin"][st["positions"]][:, None]
        x1, x2 = x[..., : d // 2], x[..., d // 2:]
        return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1)

    pool = st["pool"]
    blk, off = st["slots"] // b, st["slots"] % b
    pool[blk, 0, 0, :, off] = turn(k, st["k_norm"]).to(pool.dtype)
    pool[blk, 0, 1, :, off] = v.to(pool.dtype)
    return turn(q, st["q_norm"]), pool


def _plain_attention(st):
    """All sequences together, padded to the longest chunk and context."""
    case, n, total = st["case"], st["max_new"], st["total"]
    h, hk, d, b = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    qs = st["q_start"].long()
    s = qs.numel() - 1
    seq = torch.repeat_interleave(torch.arange(s, device=DEV), qs[1:] - qs[:-1], output_size=total)
    node = torch.arange(total, device=DEV) - qs[seq]
    pos = torch.arange(st["max_total"], device=DEV)
    blk = st["block_tables"].long()[:, pos // b]
    off = (pos % b).expand_as(blk)
    k, v = (st["pool"][blk, st["layer"], i, :, off].permute(0, 2, 1, 3).float() for i in (0, 1))
    end = (st["prefix_lens"].long() + qs[1:] - qs[:-1])[:, None]
    v = torch.where((pos < end)[:, None, :, None], v, 0.0)              # pages behind a sequence's end may hold anything
    q = torch.zeros(s, n, h, d, device=DEV)
    q[seq, node] = st["q"]
    q = q.view(s, n, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(s, hk, n * (h // hk), d)
    x = torch.matmul(q, k.transpose(2, 3)).view(s, hk, n, h // hk, -1) * (1.0 / math.sqrt(d))
    last = st["prefix_lens"].long()[:, None] + torch.arange(n, device=DEV)
    see = (pos <= last[..., None]) & (pos < end)[:, None]
    x = x.masked_fill_(~see[:, None, :, None, :], -math.inf)
    e = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    o = torch.matmul(e.view(s, hk, n * (h // hk), -1), v).view(s, hk, n, h // hk, d) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 2, 1, 3, 4).reshape(s, n, h, d)[seq, node]


def _plain_fork(st):
    pool, b = st["pool"], st["case"]["block"]
    old, lens, parents = st["block_tables"].long(), st["lens"].long(), st["parents"].long()
    s, m = old.shape
    n, nb = parents.numel(), pool.shape[0]
    me, col = torch.arange(n, device=DEV), torch.arange(m, device=DEV)
    live = parents >= 0
    p = parents.clamp(min=0)
    ln = torch.where(live, lens[p], 0)
    full, rest = ln // b, ln % b
    first = torch.full((s,), n, dtype=torch.int64, device=DEV).scatter_reduce_(0, p, torch.where(live, me, n), "amin")
    fresh = live & ((rest == 0) | (first[p] != me))
    # counts: what the old sequences hold goes, what the children share or keep comes
    shared = (col < full[:, None]) & live[:, None]
    keep = live & ~fresh
    held = (col * b < lens[:, None]).int()
    ref = st["ref_counts"].clone()
    ref.scatter_add_(0, old.reshape(-1), -held.reshape(-1))
    ref.scatter_add_(0, old[p].reshape(-1), shared.int().reshape(-1))
    ref.scatter_add_(0, old[p, full.clamp(max=m - 1)], keep.int())
    free = torch.argsort((ref > 0).int(), stable=True)                  # free pages first, lowest first
    page = torch.where(fresh, free[(fresh.cumsum(0) - 1).clamp(min=0, max=nb - 1)], old[p, full.clamp(max=m - 1)])
    ref.scatter_add_(0, page, fresh.int())
    new = torch.where(shared, old[p], 0)
    new[me, full] = torch.where(live, page, new[me, full])
    slots = torch.where(live, page * b + rest, -1)
    c = fresh & (rest > 0)
    src, dst, keep_rows = old[p, full][c], page[c], torch.arange(b, device=DEV) < rest[c][:, None]
    pool[dst] = torch.where(keep_rows[:, None, None, None, :, None], pool[src], pool[dst])
    return new.int(), ln.int(), slots, ref, pool


def _plain_compact(st):
    pool, ref = st["pool"], st["ref_counts"]
    nb = pool.shape[0]
    at = torch.arange(nb, device=DEV)
    used = ref > 0
    u = used.sum()
    src, dst = at[used & (at >= u)], at[~used & (at < u)]
    to = at.clone()
    to[src] = dst
    pool[dst] = pool[src]
    new = torch.zeros_like(ref)
    new[to[used]] = ref[used]
    return to[st["block_tables"].long()].int(), new, to.int(), u.int().view(1), pool


PLAIN = {"write": _plain_write, "attention": _plain_attention, "fork": _plain_fork, "compact": _plain_compact}


# --------------------------------------------------------------------------- #
# the framework's operators
# --------------------------------------------------------------------------- #

def _own(st):
    from kshipra_b200 import kv_cache as kv
    op = st["case"]["op"]
    if op == "write":
        q = kv.rope_cache_write(st["qkv"], st["pool"], 0, st["positions"], st["slots"], st["cos"], st["sin"],
                                q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS, out=st["out"])
        return q, st["pool"]
    if op == "attention":
        return kv.cache_attention(st["q"], st["pool"], st["layer"], st["block_tables"], st["q_start"], st["prefix_lens"],
                                  st["max_new"], st["max_total"], out=st["out"])
    if op == "fork":
        return (*kv.fork_pages(st["pool"], st["block_tables"], st["lens"], st["parents"], st["ref_counts"]), st["pool"])
    return (*kv.compact_pages(st["pool"], st["block_tables"], st["ref_counts"]), st["pool"])


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


def work(case):
    op, hk, d, b = case["op"], case["kv_heads"], case["head_dim"], case["block"]
    if op == "write":
        t, h = case["rows"], case["heads"]
        return {"bytes": t * (4.0 * (h + 2 * hk) * d + 4.0 * h * d + 4.0 * hk * d + 4.0 * d + 16), "flops": 7.0 * t * (h + hk) * d}
    if op == "attention":
        pre, new = _lens(case)
        return {"bytes": float((pre + new).sum()) * 4 * hk * d + 8.0 * float(new.sum()) * case["heads"] * d,
                "flops": 4.0 * float((new * (pre + (new + 1) / 2)).sum()) * case["heads"] * d}
    row = 4.0 * case["layers"] * hk * d                                 # K and V of a position, in all layers
    if op == "fork":
        n, m = case["seqs"] * case["beams"], case["ctx"] // b + 2
        copies = case["seqs"] * (case["beams"] - 1.0) * 0.6             # about: children that are not their parent's first
        return {"bytes": 8.0 * n * m + 2.0 * copies * row * b / 2, "flops": float(n * m)}
    moved = case["used"] * (1.0 - case["used"] / case["pages"])
    return {"bytes": 2.0 * moved * row * b + 8.0 * case["pages"], "flops": float(case["pages"])}


# --------------------------------------------------------------------------- #
# definitions in 64 bits
# --------------------------------------------------------------------------- #

def _exact_write(st):
    case = st["case"]
    h, hk, d, b = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    rows = st["qkv"].double().view(-1, h + 2 * hk, d)
    pool = st["pool"].double()
    q = torch.empty(rows.shape[0], h, d, dtype=torch.float64, device=DEV)
    cos, sin = st["cos"].double()[st["positions"]], st["sin"].double()[st["positions"]]
    for x in range(h + 2 * hk):
        r = rows[:, x]
        w = st["q_norm"] if x < h else st["k_norm"]
        if x < h + hk:
            if w is not None:
                r = r / torch.sqrt((r ** 2).sum(1, keepdim=True) / d + EPS) * w.double()
            a, c = r[:, : d // 2], r[:, d // 2:]
            r = torch.cat([a * cos - c * sin, a * sin + c * cos], 1)
        if x < h:
            q[:, x] = r
        else:
            pool[st["slots"] // b, 0, 0 if x < h + hk else 1, (x - h) % hk, st["slots"] % b] = r
    return q, pool


def _exact_attention(st):
    case, b, d = st["case"], st["case"]["block"], st["case"]["head_dim"]
    g = case["heads"] // case["kv_heads"]
    qs, pre = st["q_start"].tolist(), st["prefix_lens"].tolist()
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    for s in range(len(pre)):
        a, n = qs[s], qs[s + 1] - qs[s]
        ln = pre[s] + n
        kv = st["pool"][st["block_tables"][s, : -(-ln // b)].long(), st["layer"]]      # [blocks, 2, hk, b, d]
        hidden = torch.ones(n, ln, dtype=torch.bool, device=DEV).triu(pre[s] + 1)
        for x in range(case["kv_heads"]):
            key = kv[:, 0, x].reshape(-1, d)[:ln].double()
            val = kv[:, 1, x].reshape(-1, d)[:ln].double()
            for y in range(x * g, x * g + g):
                sc = (st["q"][a: a + n, y].double() @ key.T) / math.sqrt(d)
                out[a: a + n, y] = torch.softmax(sc.masked_fill_(hidden, -math.inf), 1) @ val
    return out


def _exact_fork(st):
    pool, b = st["pool"].double(), st["case"]["block"]
    old, lens, parents = st["block_tables"].tolist(), st["lens"].tolist(), st["parents"].tolist()
    ref = st["ref_counts"].tolist()
    m = len(old[0])
    for row, ln in zip(old, lens):
        for page in row[: -(-ln // b)]:
            ref[page] -= 1
    new, ln_out, slots, wait, seen = [], [], [], [], set()
    for i, p in enumerate(parents):
        row = [0] * m
        if p >= 0:
            full, rest = divmod(lens[p], b)
            row[:full] = old[p][:full]
            for page in row[:full]:
                ref[page] += 1
            if rest and p not in seen:
                row[full] = old[p][full]
                ref[row[full]] += 1
            else:
                wait.append((i, p, full, rest))
            seen.add(p)
        new.append(row)
        ln_out.append(lens[p] if p >= 0 else 0)
    free = iter([i for i, r in enumerate(ref) if r == 0])
    for i, p, full, rest in wait:
        page = next(free)
        new[i][full] = page
        ref[page] = 1
        pool[page, :, :, :, :rest] = pool[old[p][full], :, :, :, :rest]
    for i, p in enumerate(parents):
        slots.append(new[i][lens[p] // b] * b + lens[p] % b if p >= 0 else -1)
    return np.array(new, np.int32), np.array(ln_out, np.int32), np.array(slots, np.int64), np.array(ref, np.int32), pool


def _exact_compact(st):
    pool, ref = st["pool"].double(), st["ref_counts"].tolist()
    to, new = list(range(len(ref))), list(ref)
    u = sum(r > 0 for r in ref)
    holes = [i for i in range(u) if ref[i] == 0]
    for page in range(u, len(ref)):
        if ref[page] > 0:
            hole = holes.pop(0)
            to[page], new[hole], new[page] = hole, ref[page], 0
            pool[hole] = pool[page]
    table = [[to[x] for x in row] for row in st["block_tables"].tolist()]
    return np.array(table, np.int32), np.array(new, np.int32), np.array(to, np.int32), np.array([u], np.int32), pool


def exact(case, seed):
    st = prepare(case, seed)
    return {"write": _exact_write, "attention": _exact_attention, "fork": _exact_fork, "compact": _exact_compact}[case["op"]](st)
