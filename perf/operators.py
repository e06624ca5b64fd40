"""Cases and plain forms of the speculative-decoding operators over the paged K/V pool.

Five operators that a decode step with drafted tokens runs one after the other:

* ``tables``     block tables, row starts, positions, slots and ancestor masks from request lengths;
* ``attention``  the drafted tokens' attention: every node of a sequence's tree over the cached positions
                 and over its own ancestors in the tree;
* ``probs``      target probabilities from logits at a temperature per row;
* ``verify``     the drafted tokens against the target's (and the draft's) probabilities from given random numbers;
* ``commit``     the accepted path's K/V moved to consecutive positions, in every layer.

``run`` computes them in plain torch where ``own`` is false and through ``kshipra_b200.speculative`` where it is true.
``exact`` restates each from its definition in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #

def _attn(name, seqs, heads, kv_heads, head_dim, block, ctx, nodes, shape, ragged, layers=1):
    return dict(name=name, op="attention", seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block=block,
                ctx=ctx, nodes=nodes, shape=shape, ragged=ragged, layers=layers)


def listed():
    return [
        # one interactive request of the 0.5B shape (14 / 2 heads of 64): a 512-token prompt, four drafted tokens in a chain
        _attn("attn-1x512-chain5-h14", 1, 14, 2, 64, 16, 512, 5, "chain", False, layers=2),
        # continuous batching of the 0.5B shape: 24 requests of uneven lengths and trees, an odd block size
        _attn("attn-24x3000-tree20-h14", 24, 14, 2, 64, 24, 3000, 20, "tree", True),
        # the 8B shape's decode batch: 64 requests at context 4096, 16-node trees
        _attn("attn-64x4096-tree16-h32", 64, 32, 8, 128, 16, 4096, 16, "tree", False),
        # few long requests of the 8B heads with large trees: two tiles of query rows, keys split over the GPU
        _attn("attn-3x31000-tree61-h32", 3, 32, 8, 128, 64, 31000, 61, "tree", True),
        # one request's step: 8 nodes behind 4096 cached positions
        dict(name="tables-1x4096-tree8", op="tables", seqs=1, block=16, ctx=4096, nodes=8, shape="tree", ragged=False),
        # a full serving batch with uneven lengths and large trees
        dict(name="tables-256x8000-tree64", op="tables", seqs=256, block=16, ctx=8000, nodes=64, shape="tree", ragged=True),
        # one request: a chain of five rows over the 0.5B vocabulary
        dict(name="probs-5x151936", op="probs", rows=5, vocab=151936),
        # 64 requests of eight nodes over the 8B vocabulary
        dict(name="probs-512x128256", op="probs", rows=512, vocab=128256),
        # one request whose drafts were looked up (no draft distribution)
        dict(name="verify-1-fixed5-151936", op="verify", seqs=1, nodes=5, vocab=151936, shape="chain", draft="fixed", ragged=False),
        # 64 requests, eight-node trees drawn from a draft model
        dict(name="verify-64-drawn8-128256", op="verify", seqs=64, nodes=8, vocab=128256, shape="tree", draft="drawn", ragged=False),
        # one request of the 0.5B shape: 24 layers
        dict(name="commit-1x24-h2x64", op="commit", seqs=1, layers=24, kv_heads=2, head_dim=64, block=16, ctx=40, nodes=8, ragged=False),
        # 48 requests of the 8B shape: 32 layers
        dict(name="commit-48x32-h8x128", op="commit", seqs=48, layers=32, kv_heads=8, head_dim=128, block=16, ctx=50, nodes=16, ragged=True),
    ]


HEADS = [(14, 2, 64), (32, 8, 128), (4, 2, 64), (16, 4, 128), (8, 2, 128), (8, 8, 64), (16, 2, 128)]
VOCABS = [1024, 151936, 128256, 32000, 50257]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["attention", "attention", "tables", "probs", "verify", "commit"])
    if op == "attention":
        h, hk, d = rng.choice(HEADS)
        return dict(op=op, seqs=_log(rng, 1, 64), heads=h, kv_heads=hk, head_dim=d, block=rng.choice([16, 24, 64, 10]),
                    ctx=_log(rng, 60, 31000), nodes=_log(rng, 1, 64), shape=rng.choice(["chain", "tree"]), ragged=rng.random() < 0.7,
                    layers=rng.choice([1, 2]))
    if op == "tables":
        return dict(op=op, seqs=_log(rng, 1, 256), block=rng.choice([16, 24, 64, 10]), ctx=_log(rng, 10, 8000), nodes=_log(rng, 1, 64),
                    shape=rng.choice(["chain", "tree"]), ragged=rng.random() < 0.7)
    if op == "probs":
        return dict(op=op, rows=_log(rng, 1, 512), vocab=rng.choice(VOCABS) + rng.choice([0, 0, 1, 3]))
    if op == "verify":
        return dict(op=op, seqs=_log(rng, 1, 64), nodes=_log(rng, 1, 16), vocab=rng.choice(VOCABS) + rng.choice([0, 0, 1]),
                    shape=rng.choice(["chain", "tree"]), draft=rng.choice(["drawn", "fixed", "greedy"]), ragged=rng.random() < 0.5)
    h, hk, d = rng.choice(HEADS)
    return dict(op=op, seqs=_log(rng, 1, 48), layers=rng.choice([2, 24, 32]), kv_heads=hk, head_dim=d, block=rng.choice([16, 24, 64]),
                ctx=_log(rng, 4, 60), nodes=_log(rng, 2, 16), ragged=rng.random() < 0.7)


def _size(case):
    """What a pass and its preparation touch, in bytes, for the bound on drawn cases."""
    w = work(case)["bytes"]
    if case["op"] == "verify":
        w = max(w, 8.0 * case["seqs"] * case["nodes"] * case["vocab"])
    if case["op"] == "attention":
        w = max(w, 8.0 * case["seqs"] * (case["ctx"] + case["nodes"]) * case["kv_heads"] * case["head_dim"] * case["layers"])
        w = max(w, 12.0 * case["seqs"] * (case["ctx"] + case["nodes"]) * case["heads"] * case["nodes"])
    if case["op"] == "commit":
        w = 8.0 * case["seqs"] * (case["ctx"] + case["nodes"] + 2 * case["block"]) * case["layers"] * case["kv_heads"] * case["head_dim"]
    return w


def draw(rng):
    most = max(_size(c) for c in listed())
    while True:
        c = _draw(rng)
        if _size(c) <= most:
            return c


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #

def _lens(case):
    """Cached positions and new nodes of each sequence, from the case alone."""
    s, n, ctx = case["seqs"], case["nodes"], case.get("ctx", 0)
    if not case["ragged"]:
        return np.full(s, ctx, np.int64), np.full(s, n, np.int64)
    r = np.random.RandomState((s * 7919 + ctx * 31 + n * 17) % (1 << 31))
    pre = r.randint(ctx // 3, ctx + 1, s)
    new = r.randint((n + 1) // 2, n + 1, s)
    pre[0], new[0] = ctx, n
    return pre.astype(np.int64), new.astype(np.int64)


def _parents(case, new, rs):
    """Parent of each node (of its own sequence, -1 for the root), in node order."""
    out = []
    for n in new:
        if case.get("shape") == "chain":
            out.append(np.arange(-1, n - 1))
        else:  # a few children a node, some chains
            out.append(np.array([-1] + [i - 1 if rs.rand() < 0.4 else rs.randint(0, i) for i in range(1, n)]))
    return np.concatenate(out)


def _blocks(pre, new, block, rs, spare):
    """Physical blocks of each sequence, shuffled over the pool: (flat ids, starts, blocks of the pool)."""
    need = -(-(pre + new) // block)
    start = np.concatenate([[0], np.cumsum(need)])
    nb = int(start[-1]) + spare
    return rs.permutation(nb)[: int(start[-1])], start, nb


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to(device=DEV, dtype=dtype)


def _table(ids, start):
    rows = [ids[a:b] for a, b in zip(start[:-1], start[1:])]
    t = np.zeros((len(rows), max(len(r) for r in rows)), np.int64)
    for i, r in enumerate(rows):
        t[i, : len(r)] = r
    return t


def _masks(parents, new, words):
    """Ancestor mask of each node, itself included, as 64-bit words."""
    out, at = np.zeros((int(new.sum()), words), np.uint64), 0
    for n in new:
        for i in range(n):
            p = parents[at + i]
            if p >= 0:
                out[at + i] = out[at + p]
            out[at + i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
        at += n
    return out.view(np.int64)


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    op = case["op"]
    st = {"case": case}
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device=DEV)  # noqa: E731
    if op == "probs":
        st["logits"] = _logits(case["rows"], case["vocab"], g)
        t = 0.5 + rand(case["rows"])
        t[rs.randint(0, case["rows"])] = 0.0 if case["rows"] > 4 else 1.0      # one greedy request among the sampled ones
        st["temperature"] = t
        st["out"] = torch.empty_like(st["logits"])
        return st
    pre, new = _lens(case)
    qs = np.concatenate([[0], np.cumsum(new)])
    st["q_start"] = _dev(qs, torch.int32)
    st["total"], st["max_nodes"] = int(qs[-1]), int(new.max())
    if op == "verify":
        par = _parents(case, new, rs)
        st["parents"] = _dev(par, torch.int32)
        _prepare_verify(st, case, new, qs, par, g, rs)
        return st
    # the tables' case names blocks of a large pool that it does not touch
    ids, start, nb = _blocks(pre, new, case["block"], rs, 509 if op == "tables" else 3)
    st["prefix_lens"] = _dev(pre, torch.int32)
    if op == "tables":
        st["new_lens"] = _dev(new, torch.int32)
        st["parents"] = _dev(_parents(case, new, rs), torch.int32)
        st["block_ids"], st["block_start"] = _dev(ids, torch.int32), _dev(start, torch.int32)
        st["max_blocks"] = int(np.diff(start).max())
        return st
    st["block_tables"] = _dev(_table(ids, start), torch.int32)
    hk, d, layers = case["kv_heads"], case["head_dim"], case["layers"]
    st["pool"] = randn(nb, layers, 2, hk, case["block"], d)
    if op == "attention":
        st["layer"] = layers - 1
        # after the rotation queries are larger than keys in trained models: scores spread over several units
        st["q"] = randn(st["total"], case["heads"], d) * 2.0
        words = -(-st["max_nodes"] // 64)
        st["mask"] = _dev(_masks(_parents(case, new, rs), new, words), torch.int64)
        st["max_total"] = int((pre + new).max())
        st["out"] = torch.empty_like(st["q"])
        return st
    # commit: a root and a random increasing path behind it
    path = np.full((case["seqs"], st["max_nodes"]), -1, np.int64)
    ln = np.zeros(case["seqs"], np.int64)
    for s, n in enumerate(new):
        k = min(int(n), 1 + int(rs.geometric(0.3)))
        path[s, :k] = np.concatenate([[0], 1 + np.sort(rs.permutation(int(n) - 1)[: k - 1])])
        ln[s] = k
    st["path"], st["path_len"] = _dev(path, torch.int32), _dev(ln, torch.int32)
    return st


def _logits(rows, vocab, g):
    """A few likely tokens over a long tail, as a language model's logits have them."""
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.0
    at = torch.randint(0, vocab, (rows, 8), generator=g, device=DEV)
    return x.scatter(1, at, 8.0 + 8.0 * torch.rand(rows, 8, generator=g, device=DEV))


def _prepare_verify(st, case, new, qs, par, g, rs):
    rows, v, total = int(qs[-1]), case["vocab"], st["total"]
    first = np.repeat(qs[:-1], new)                       # first row of each node's sequence
    up = _dev(np.where(par >= 0, par, 0) + first, torch.int64)   # row of each node's parent
    x = _logits(rows, v, g)
    st["u_accept"] = torch.rand(total, generator=g, device=DEV)
    st["u_sample"] = torch.rand(len(new), generator=g, device=DEV)
    if case["draft"] == "greedy":
        st["target_tokens"] = x.argmax(1)
        hit = torch.rand(total, generator=g, device=DEV) < 0.7
        st["tokens"] = torch.where(hit, st["target_tokens"][up], torch.randint(0, v, (total,), generator=g, device=DEV))
        return
    st["target_probs"] = torch.softmax(x, 1)
    x += 0.7 * torch.randn(rows, v, generator=g, device=DEV)    # the draft model: near the target
    if case["draft"] == "drawn":
        st["draft_probs"] = torch.softmax(x, 1)
        st["tokens"] = torch.multinomial(st["draft_probs"][up], 1, generator=g).view(-1)
    else:                                                 # the node's k-th child carries the k-th likely token
        rank, seen = np.zeros(rows, np.int64), {}
        for i in range(rows):
            key = (int(first[i]), int(par[i]))
            rank[i] = min(seen.get(key, 0), 63)
            seen[key] = rank[i] + 1
        st["tokens"] = x.topk(64, 1).indices[up, _dev(rank, torch.int64)]


# --------------------------------------------------------------------------- #
# plain forms
# --------------------------------------------------------------------------- #

def _plain_tables(st):
    case = st["case"]
    b, n, total = case["block"], st["max_nodes"], st["total"]
    new, pre, par = st["new_lens"].long(), st["prefix_lens"].long(), st["parents"].long()
    s = new.numel()
    qs = torch.zeros(s + 1, dtype=torch.int64, device=DEV)
    qs[1:] = new.cumsum(0)
    seq = torch.repeat_interleave(torch.arange(s, device=DEV), new, output_size=total)
    node = torch.arange(total, device=DEV) - qs[seq]
    bs = st["block_start"].long()
    at = bs[:-1, None] + torch.arange(st["max_blocks"], device=DEV)
    table = torch.where(at < bs[1:, None], st["block_ids"].long()[at.clamp(max=st["block_ids"].numel() - 1)], 0)
    # ancestors: the closure of "is itself or its parent" by squaring
    anc = torch.zeros(s, n, n, device=DEV)
    anc[seq, node, node] = 1.0
    anc[seq, node, torch.where(par >= 0, par, node)] = 1.0
    for _ in range(max(1, (n - 1).bit_length())):
        anc = (torch.matmul(anc, anc) > 0).float()
    rows = anc[seq, node]                                             # [T, n]
    pos = pre[seq] + rows.sum(1).long() - 1
    at = pre[seq] + node
    slots = table[seq, at // b] * b + at % b
    words = -(-n // 64)
    bits = torch.zeros(total, words * 64, dtype=torch.int64, device=DEV)
    bits[:, :n] = rows.long()
    mask = (bits.view(total, words, 64) << torch.arange(64, device=DEV)).sum(2)
    return qs.int(), table.int(), pos, slots, mask


def _gather(st):
    """K and V of every sequence's positions [S, hkv, max_total, d], and who may see them [S, n, max_total]."""
    pool, b, layer = st["pool"], st["case"]["block"], st["layer"]
    pos = torch.arange(st["max_total"], device=DEV)
    blk = st["block_tables"].long()[:, pos // b]
    off = (pos % b).expand_as(blk)
    k = pool[:, layer, 0][blk, :, off].permute(0, 2, 1, 3)
    v = pool[:, layer, 1][blk, :, off].permute(0, 2, 1, 3)
    return k, v, pos


def _plain_attention(st):
    case, n, total = st["case"], st["max_nodes"], st["total"]
    h, hk, d = case["heads"], case["kv_heads"], case["head_dim"]
    qs = st["q_start"].long()
    s = qs.numel() - 1
    seq = torch.repeat_interleave(torch.arange(s, device=DEV), qs[1:] - qs[:-1], output_size=total)
    node = torch.arange(total, device=DEV) - qs[seq]
    k, v, pos = _gather(st)
    q = torch.zeros(s, n, h, d, device=DEV)
    q[seq, node] = st["q"]
    q = q.view(s, n, hk, h // hk, d).permute(0, 2, 1, 3, 4).reshape(s, hk, n * (h // hk), d)
    bits = torch.zeros(s, n, st["mask"].shape[1], dtype=torch.int64, device=DEV)
    bits[seq, node] = st["mask"]
    pre = st["prefix_lens"].long()[:, None]
    rel = pos - pre                                                   # [S, max_total] node index of each position
    inside = (rel >= 0) & (rel < (qs[1:] - qs[:-1])[:, None])
    r = torch.where(inside, rel, 0)
    word = torch.gather(bits, 2, (r >> 6)[:, None, :].expand(s, n, -1))
    see = (rel < 0)[:, None, :] | (inside[:, None, :] & (((word >> (r & 63)[:, None, :]) & 1) != 0))
    x = torch.matmul(q, k.transpose(2, 3)).view(s, hk, n, h // hk, -1) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~see[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    e = torch.exp(x - m)
    o = torch.matmul(e.view(s, hk, n * (h // hk), -1), v).view(s, hk, n, h // hk, d) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.permute(0, 2, 1, 3, 4).reshape(s, n, h, d)[seq, node]


def _plain_probs(st):
    x, t = st["logits"], st["temperature"][:, None]
    z = x / torch.where(t > 0, t, 1.0)
    e = torch.exp(z - z.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    hot = torch.zeros_like(x).scatter_(1, x.argmax(1, keepdim=True), 1.0)
    return torch.where(t > 0, p, hot)


def _plain_verify(st):
    """All sequences together, node after node.  Sums over the vocabulary are held in 64 bits: the choice of a
    token is a whole number and may not depend on the order of a sum."""
    case, n = st["case"], st["max_nodes"]
    qs = st["q_start"].long()
    s = qs.numel() - 1
    dev = torch.arange(s, device=DEV)
    count = qs[1:] - qs[:-1]
    cur = torch.zeros(s, dtype=torch.int64, device=DEV)
    path = torch.full((s, n), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    length = torch.ones(s, dtype=torch.int64, device=DEV)
    greedy, drawn = "target_tokens" in st, "draft_probs" in st
    if not greedy:
        r = st["target_probs"][qs[:-1]].double()
        z = torch.ones(s, dtype=torch.float64, device=DEV)
    for i in range(1, n):
        row = qs[:-1] + i
        row = torch.where(i < count, row, qs[:-1])
        mine = (i < count) & (st["parents"].long()[row] == cur)
        tok = st["tokens"][row]
        if greedy:
            yes = mine & (tok == st["target_tokens"][qs[:-1] + cur])
        else:
            u = st["u_accept"][row].double()
            q = st["draft_probs"][qs[:-1] + cur].double() if drawn else None
            at = q[dev, tok] if drawn else 1.0
            yes = mine & (u * z * at < r[dev, tok])
            no = mine & ~yes
            if drawn:
                left = (r - z[:, None] * q).clamp(min=0)
                r = torch.where(no[:, None], left, r)
                z = torch.where(no, left.sum(1), z)
            else:
                gone = r[dev, tok]
                z = torch.where(no, z - gone, z)
                r[dev, tok] = torch.where(no, 0.0, gone)
            r = torch.where(yes[:, None], st["target_probs"][row].double(), r)
            z = torch.where(yes, 1.0, z)
        cur = torch.where(yes, i, cur)
        path[dev, length.clamp(max=n - 1)] = torch.where(yes, i, path[dev, length.clamp(max=n - 1)].long()).int()
        length = length + yes.long()
    if greedy:
        return path, length.int(), st["target_tokens"][qs[:-1] + cur]
    r = torch.where((r.sum(1) > 0)[:, None], r, st["target_probs"][qs[:-1] + cur].double())
    c = r.cumsum(1)
    over = c > st["u_sample"].double()[:, None] * c[:, -1:]
    return path, length.int(), over.to(torch.int8).argmax(1)


def _plain_commit(st):
    pool, b, n = st["pool"], st["case"]["block"], st["max_nodes"]
    pre, path = st["prefix_lens"].long()[:, None], st["path"].long()
    j = torch.arange(n, device=DEV)
    on = (j < st["path_len"].long()[:, None]) & (path != j)
    src, dst = (pre + path)[on], (pre + j)[on]
    t = st["block_tables"].long()
    seq = torch.arange(t.shape[0], device=DEV)[:, None].expand_as(on)[on]
    pool[t[seq, dst // b], :, :, :, dst % b] = pool[t[seq, src // b], :, :, :, src % b]
    return pool, (st["prefix_lens"] + st["path_len"]).int()


PLAIN = {"tables": _plain_tables, "attention": _plain_attention, "probs": _plain_probs, "verify": _plain_verify, "commit": _plain_commit}


# --------------------------------------------------------------------------- #
# the framework's operators
# --------------------------------------------------------------------------- #

def _own(st):
    from kshipra_b200 import speculative as sp
    op = st["case"]["op"]
    if op == "tables":
        return sp.tree_tables(st["prefix_lens"], st["new_lens"], st["total"], st["case"]["block"], st["max_nodes"], st["max_blocks"],
                              block_ids=st["block_ids"], block_start=st["block_start"], parents=st["parents"])
    if op == "attention":
        return sp.tree_attention(st["q"], st["pool"], st["layer"], st["block_tables"], st["q_start"], st["prefix_lens"], st["mask"],
                                 st["max_nodes"], st["max_total"], out=st["out"])
    if op == "probs":
        return sp.target_probs(st["logits"], st["temperature"], out=st["out"])
    if op == "verify":
        return sp.verify_tree(st["tokens"], st["parents"], st["q_start"], st["max_nodes"], target_probs=st.get("target_probs"),
                              draft_probs=st.get("draft_probs"), target_tokens=st.get("target_tokens"), u_accept=st["u_accept"],
                              u_sample=st["u_sample"])
    return st["pool"], sp.commit_tree(st["pool"], st["block_tables"], st["prefix_lens"], st["path"], st["path_len"])


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "probs":
        return {"bytes": 8.0 * case["rows"] * case["vocab"], "flops": 4.0 * case["rows"] * case["vocab"]}
    pre, new = _lens(case)
    s, t = case["seqs"], float(new.sum())
    if op == "verify":
        if case["draft"] == "greedy":
            return {"bytes": 20.0 * t + 20.0 * s, "flops": t}
        rows = 2.0 if case["draft"] == "drawn" else 1.0
        return {"bytes": 4.0 * rows * s * case["vocab"] + 28.0 * t, "flops": 2.0 * rows * s * case["vocab"]}
    if op == "tables":
        need = -(-(pre + new) // case["block"])
        words = -(-int(new.max()) // 64)
        return {"bytes": float(4 * need.sum() + 4 * s * need.max() + 16 * s) + t * (4 + 16 + 8 * words), "flops": 4.0 * t}
    if op == "attention":
        kv = float((pre + new).sum()) * 2 * case["kv_heads"] * case["head_dim"] * 4
        return {"bytes": kv + 8.0 * t * case["heads"] * case["head_dim"],
                "flops": 4.0 * float((new * (pre + (new + 1) / 2)).sum()) * case["heads"] * case["head_dim"]}
    # about 1 / 0.3 nodes of a path besides the root, most of them not in place
    moved = float(np.minimum(new - 1, 1.0 / 0.3).sum())
    return {"bytes": 2.0 * moved * case["layers"] * 2 * case["kv_heads"] * case["head_dim"] * 4, "flops": moved}


# --------------------------------------------------------------------------- #
# definitions in 64 bits
# --------------------------------------------------------------------------- #

def _exact_tables(st):
    b = st["case"]["block"]
    new, pre, par = (st[k].cpu().numpy().astype(np.int64) for k in ("new_lens", "prefix_lens", "parents"))
    ids, start = st["block_ids"].cpu().numpy(), st["block_start"].cpu().numpy()
    qs = [0]
    table = np.zeros((len(new), st["max_blocks"]), np.int32)
    pos, slots = [], []
    for s, n in enumerate(new):
        mine = ids[start[s]: start[s + 1]]
        table[s, : len(mine)] = mine
        depth = []
        for i in range(n):
            p = par[qs[-1] + i]
            depth.append(0 if p < 0 else depth[p] + 1)
            pos.append(pre[s] + depth[i])
            slots.append(int(mine[(pre[s] + i) // b]) * b + (pre[s] + i) % b)
        qs.append(qs[-1] + int(n))
    mask = _masks(par, new, -(-st["max_nodes"] // 64))
    return np.array(qs, np.int32), table, np.array(pos, np.int64), np.array(slots, np.int64), mask


def _exact_attention(st):
    case, b, d = st["case"], st["case"]["block"], st["case"]["head_dim"]
    h, hk = case["heads"], case["kv_heads"]
    g = h // hk
    qs, pre = st["q_start"].tolist(), st["prefix_lens"].tolist()
    masks = st["mask"].cpu().numpy().view(np.uint64)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEV)
    for s in range(len(pre)):
        a, n = qs[s], qs[s + 1] - qs[s]
        ln = pre[s] + n
        used = st["block_tables"][s, : -(-ln // b)].long()
        kv = st["pool"][used, st["layer"]]                              # [blocks, 2, hk, b, d]
        hidden = np.ones((n, ln), bool)
        hidden[:, : pre[s]] = False
        for i in range(n):
            for j in range(n):
                hidden[i, pre[s] + j] = not (int(masks[a + i, j // 64]) >> (j % 64)) & 1
        hidden = torch.from_numpy(hidden).to(DEV)
        for x in range(hk):
            key = kv[:, 0, x].reshape(-1, d)[:ln].double()
            val = kv[:, 1, x].reshape(-1, d)[:ln].double()
            for y in range(x * g, x * g + g):
                sc = (st["q"][a: a + n, y].double() @ key.T) / math.sqrt(d)
                sc[hidden] = -math.inf
                out[a: a + n, y] = torch.softmax(sc, 1) @ val
    return out


def _exact_probs(st):
    out = torch.empty(st["logits"].shape, dtype=torch.float64, device=DEV)
    for i, t in enumerate(st["temperature"].tolist()):
        x = st["logits"][i].double()
        if t > 0:
            out[i] = torch.softmax(x / t, 0)
        else:
            out[i] = 0.0
            out[i, int(x.argmax())] = 1.0
    return out


def _exact_verify(st):
    n = st["max_nodes"]
    qs, par, tok = st["q_start"].tolist(), st["parents"].tolist(), st["tokens"].tolist()
    uq, us = st["u_accept"].double().tolist(), st["u_sample"].double().tolist()
    path, lens, nxt = np.full((len(us), n), -1, np.int32), np.zeros(len(us), np.int32), np.zeros(len(us), np.int64)
    row = lambda t, i: t[i].cpu().numpy().astype(np.float64)  # noqa: E731
    for s, (a, e) in enumerate(zip(qs[:-1], qs[1:])):
        cur, took = 0, [0]
        if "target_tokens" in st:
            want = st["target_tokens"][a:e].tolist()
            for i in range(1, e - a):
                if par[a + i] == cur and tok[a + i] == want[cur]:
                    cur = i
                    took.append(i)
            nxt[s] = want[cur]
        else:
            r, z = row(st["target_probs"], a), 1.0
            q = row(st["draft_probs"], a) if "draft_probs" in st else None
            for i in range(1, e - a):
                if par[a + i] != cur:
                    continue
                t = tok[a + i]
                if uq[a + i] * z * (1.0 if q is None else q[t]) < r[t]:
                    cur = i
                    took.append(i)
                    r, z = row(st["target_probs"], a + i), 1.0
                    q = row(st["draft_probs"], a + i) if "draft_probs" in st else None
                elif q is None:
                    z -= r[t]
                    r[t] = 0.0
                else:
                    r = np.maximum(r - z * q, 0.0)
                    z = math.fsum(r)
            if not r.any():
                r = row(st["target_probs"], a + cur)
            c = np.cumsum(r)
            nxt[s] = int(np.argmax(c > us[s] * c[-1]))
        path[s, : len(took)] = took
        lens[s] = len(took)
    return path, lens, nxt


def _exact_commit(st):
    pool, b = st["pool"].double(), st["case"]["block"]
    pre, path, ln = st["prefix_lens"].tolist(), st["path"].tolist(), st["path_len"].tolist()
    table = st["block_tables"].tolist()
    for s in range(len(pre)):
        for j in range(ln[s]):
            x, y = pre[s] + path[s][j], pre[s] + j
            if x != y:
                pool[table[s][y // b], :, :, :, y % b] = pool[table[s][x // b], :, :, :, x % b]
    return pool, np.array(pre, np.int32) + np.array(ln, np.int32)


def exact(case, seed):
    st = prepare(case, seed)
    return {"tables": _exact_tables, "attention": _exact_attention, "probs": _exact_probs, "verify": _exact_verify,
            "commit": _exact_commit}[case["op"]](st)
