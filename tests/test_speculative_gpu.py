"""Speculative-decoding operators on the GPU against plain implementations in
64 bits, and the decoder against ``generate``.

Tolerances: tables, verification and the K/V move are exact.  Attention: the
framework's bound for its fp32 attention, a relative L2 error of 1e-5 against
64 bits; single elements within 8e-5 of the largest value the row can reach
(scores of size 16 held to 2^-22 relative move a probability by 16 * 2^-22 =
4e-6, and an output is a mean of values with such weights; the factor 20 is for
rows of few keys).  Probabilities: expf is good to 2 ulp, the argument (x -
max) / T to 1.5 ulp of at most 40 in size (40 * 1.5 * 2^-24 = 3.6e-6), the sum
to 1e-6: 1e-5 relative.
"""

import numpy as np
import pytest
import torch

from kshipra_b200 import _lib
from kshipra_b200 import speculative as sp

pytestmark = pytest.mark.gpu

BAD_BLOCK, BAD_TOKEN, BAD_LENGTH, BAD_PARENT, BAD_PROBS = 2, 16, 32, 128, 256


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def new_flags():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def trees(lens, rs, chain=False):
    return [np.arange(-1, n - 1) if chain else
            np.array([-1] + [int(rs.randint(max(0, i - 5), i)) for i in range(1, n)], np.int64)[:n]
            for n in lens]


def ancestors(par):
    see = np.zeros((len(par), len(par)), bool)
    for i, p in enumerate(par):
        if 0 <= p < i:
            see[i] = see[p]
        see[i, i] = True
    return see


def pack(see, words):
    out = np.zeros((see.shape[0], words), np.uint64)
    for i, j in zip(*np.nonzero(see)):
        out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


# --------------------------------------------------------------------------- #
# tables
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("block", [1, 7, 16, 64])
@pytest.mark.parametrize("lens", [[1], [5, 0, 3], [64, 1, 33, 64], [65, 200, 256], [1] * 300])
@pytest.mark.parametrize("chain", [True, False])
def test_tree_tables(block, lens, chain):
    rs = np.random.RandomState(len(lens) * 100 + block)
    pre = rs.randint(0, 200, len(lens))
    par = trees(lens, rs, chain)
    need = [-(-(p + n) // block) for p, n in zip(pre, lens)]
    start = np.concatenate([[0], np.cumsum(need)])
    ids = rs.permutation(int(start[-1]) + 5)[:start[-1]]
    most, T = max(lens), sum(lens)
    flags = new_flags()
    qs, bt, pos, slots, mask = sp.tree_tables(
        i32(pre), i32(lens), T, block, most, max(need), block_ids=i32(ids),
        block_start=i32(start), parents=i32(np.concatenate(par)), flags=flags)
    assert int(flags) == 0
    words = -(-most // 64)
    np.testing.assert_array_equal(qs.cpu(), np.concatenate([[0], np.cumsum(lens)]))
    for s, n in enumerate(lens):
        mine = ids[start[s]:start[s + 1]]
        np.testing.assert_array_equal(bt[s].cpu(), np.pad(mine, (0, max(need) - need[s])))
        a = int(qs[s])
        see = ancestors(par[s])
        at = pre[s] + np.arange(n)
        np.testing.assert_array_equal(pos[a:a + n].cpu(), pre[s] + see.sum(1) - 1)
        np.testing.assert_array_equal(slots[a:a + n].cpu(), mine[at // block] * block + at % block)
        np.testing.assert_array_equal(mask[a:a + n].cpu(), pack(see, words))
    # ready tables and plain chunks
    qs2, bt2, pos2, slots2, none = sp.tree_tables(i32(pre), i32(lens), T, block, most, max(need),
                                                  block_tables=bt, flags=flags)
    assert none is None and bt2 is bt and int(flags) == 0
    assert torch.equal(qs, qs2) and torch.equal(slots, slots2)
    np.testing.assert_array_equal(pos2.cpu(), np.concatenate(
        [p + np.arange(n) for p, n in zip(pre, lens)]))


def test_tree_tables_long_chunks():
    pre, lens = [0, 17], [1000, 3000]
    bt = torch.arange(2 * 200, dtype=torch.int32, device="cuda").view(2, 200)
    qs, _, pos, slots, _ = sp.tree_tables(i32(pre), i32(lens), 4000, 16, 3000, 200, block_tables=bt)
    want = np.concatenate([np.arange(1000), 17 + np.arange(3000)])
    np.testing.assert_array_equal(pos.cpu(), want)
    np.testing.assert_array_equal(slots.cpu(), want + np.repeat([0, 3200], lens))


def test_tree_tables_reports_bad_input():
    ids, start = i32([3, 4]), i32([0, 1, 2])
    args = dict(block_ids=ids, block_start=start)
    # a parent that is no earlier node counts as a root
    flags = new_flags()
    _, _, pos, _, mask = sp.tree_tables(i32([2, 0]), i32([3, 1]), 4, 16, 3, 1,
                                        parents=i32([-1, 2, 0, 0]), flags=flags, **args)
    assert int(flags) == BAD_PARENT
    assert pos.tolist() == [2, 2, 3, 0] and mask.view(-1).tolist() == [1, 2, 5, 1]
    # past its blocks; lengths that do not add up; negative lengths
    for pre, new, total in (([15, 0], [3, 1], 4), ([0, 0], [3, 1], 6), ([0, 0], [3, 1], 3),
                            ([-1, 0], [3, 1], 4), ([0, 0], [-3, 1], 1)):
        flags = new_flags()
        _, _, pos, slots, _ = sp.tree_tables(i32(pre), i32(new), total, 16, 3, 1, flags=flags,
                                             parents=i32([-1, 0, 0, -1, -1, -1][:total]), **args)
        assert int(flags) & BAD_LENGTH
        if total == 6:
            assert pos.tolist()[4:] == [0, 0] and slots.tolist()[4:] == [-1, -1]
        if pre[0] == 15:
            assert slots.tolist()[:3] == [3 * 16 + 15, -1, -1]
    flags = new_flags()
    sp.tree_tables(i32([0, 0]), i32([1, 1]), 2, 16, 1, 1, block_ids=ids, block_start=i32([0, 1, 9]),
                   flags=flags)
    assert int(flags) == BAD_LENGTH


# --------------------------------------------------------------------------- #
# attention
# --------------------------------------------------------------------------- #

class Case:
    """A batch with shuffled blocks; whatever no node may see is NaN."""

    def __init__(self, pre, lens, hq, hkv, d, block, seed=0, layers=2, chain=False, scale=(1.0, 1.0),
                 see=None):
        rs = np.random.RandomState(seed)
        g = torch.Generator().manual_seed(seed)
        self.pre, self.lens, self.block = list(pre), list(lens), block
        need = [max(1, -(-(p + n) // block)) for p, n in zip(pre, lens)]
        nb = sum(need) + 2
        order = rs.permutation(nb)
        self.layer = layers - 1
        self.pool = torch.full((nb, layers, 2, hkv, block, d), float("nan"))
        self.bt = np.zeros((len(lens), max(need)), np.int64)
        self.kv = []
        at = 0
        for s, (p, n) in enumerate(zip(pre, lens)):
            self.bt[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            kv = torch.randn((2, hkv, p + n, d), generator=g) + 0.3
            kv[0] *= scale[0]
            kv[1] *= scale[1]
            self.kv.append(kv)
            for t in range(p + n):
                self.pool[self.bt[s, t // block], self.layer, :, :, t % block] = kv[:, :, t]
        self.q = torch.randn((sum(lens), hq, d), generator=g) * (2.0 / scale[0])
        self.see = see if see is not None else [ancestors(p) for p in trees(lens, rs, chain)]
        self.words = max(1, -(-max(lens) // 64))
        self.mask = torch.from_numpy(np.concatenate([pack(x, self.words) for x in self.see]))
        self.qs = np.concatenate([[0], np.cumsum(lens)])

    def run(self, mask=True, flags=None, **kw):
        flags = new_flags() if flags is None else flags
        out = sp.tree_attention(self.q.cuda(), self.pool.cuda(), self.layer, i32(self.bt),
                                i32(self.qs), i32(self.pre), self.mask.cuda() if mask else None,
                                max(self.lens), max(p + n for p, n in zip(self.pre, self.lens)),
                                flags=flags, **kw)
        return out.cpu(), int(flags)

    def plain(self):
        T, hq, d = self.q.shape
        out = torch.zeros((T, hq, d), dtype=torch.float64)
        for s, (p, n) in enumerate(zip(self.pre, self.lens)):
            kv = self.kv[s].double()
            g = hq // kv.shape[1]
            for i in range(n):
                on = np.concatenate([np.ones(p, bool), self.see[s][i]])
                if not on.any():
                    continue
                k, v = kv[0][:, on], kv[1][:, on]
                for h in range(hq):
                    x = k[h // g] @ self.q[self.qs[s] + i, h].double() / d ** 0.5
                    out[self.qs[s] + i, h] = torch.softmax(x, 0) @ v[h // g]
        return out

    def check(self, got=None, rel=1e-5, top_rel=8e-5):
        if got is None:
            got, f = self.run()
            assert f == 0
        want = self.plain()
        assert torch.equal(torch.isfinite(got), torch.isfinite(want))
        err = (got.double() - want).norm() / want.norm().clamp(min=1e-30)
        assert err <= rel, float(err)
        top = max(float(kv[1].abs().max()) for kv in self.kv if kv.numel())
        assert (got.double() - want).abs().max() <= top_rel * top
        return got


SHAPES = [(14, 2, 64), (32, 8, 128), (4, 4, 64), (8, 1, 128), (6, 2, 80), (3, 3, 32), (2, 1, 256)]


@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("pre,lens", [([0], [1]), ([1], [1]), ([63], [2]), ([64, 0, 7], [5, 9, 1]),
                                      ([130, 61], [33, 3])])
def test_tree_attention_shapes(hq, hkv, d, pre, lens):
    Case(pre, lens, hq, hkv, d, 16, seed=d + len(pre)).check()


@pytest.mark.parametrize("block", [1, 7, 16, 24, 64, 100])
def test_tree_attention_blocks_end_inside_tiles(block):
    Case([200, 67, 129], [10, 16, 7], 8, 2, 128, block, seed=block).check()
    Case([200, 67, 129], [10, 16, 7], 14, 2, 64, block, seed=block).check()


@pytest.mark.parametrize("lens", [[64], [65, 3], [200, 1], [256]])
def test_tree_attention_large_trees(lens):
    Case([77] * len(lens), lens, 8, 2, 64, 16, seed=lens[0]).check()
    Case([40] * len(lens), lens, 4, 1, 128, 16, seed=lens[0]).check()


def test_tree_attention_long_context_and_many_sequences():
    Case([3000, 5, 1100], [4, 6, 3], 4, 2, 128, 16, seed=3).check()
    rs = np.random.RandomState(5)
    Case(rs.randint(0, 300, 70), rs.randint(1, 9, 70), 4, 2, 64, 16, seed=4).check()


def test_tree_attention_sequences_without_nodes():
    Case([10, 50, 0, 20], [3, 0, 2, 0], 4, 2, 64, 16, seed=9).check()


@pytest.mark.parametrize("d", [64, 128])
def test_tree_attention_of_tensors_off_16_byte_boundaries(d):
    """The same call on a pool, a q or an out that starts in the middle of 16 bytes."""
    c = Case([70, 3], [9, 4], 4, 2, d, 16, seed=d)
    want = c.check()

    def off(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1).cuda()
        return buf[1:].view(t.shape)

    q, pool, out = c.q.cuda(), c.pool.cuda(), torch.empty_like(c.q, device="cuda")
    rest = [c.layer, i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda(), 9, 79]
    for args, o in (((off(q), pool), out), ((q, off(pool)), out), ((q, pool), off(out))):
        assert sum(t.data_ptr() % 16 for t in (*args, o)) == 4
        got = sp.tree_attention(*args, *rest, out=o).cpu()
        c.check(got)
        assert ((got - want).norm() / want.norm()) <= 2e-5


def test_tree_attention_without_mask_is_causal():
    c = Case([50, 3], [20, 70], 8, 2, 64, 16, seed=1, chain=True)
    got, f = c.run(mask=False)
    assert f == 0
    c.check(got)


def test_tree_attention_empty_rows_and_odd_masks():
    """Masks that are no tree: nodes that see nothing, only later nodes, or all."""
    rs = np.random.RandomState(2)
    see = [np.zeros((6, 6), bool), rs.rand(70, 70) < 0.1]
    see[0][1] = True
    see[0][2, 5] = True
    see[1][3] = False
    c = Case([0, 0], [6, 70], 4, 2, 128, 16, seed=2, see=see)
    got = c.check()
    assert (got[0] == 0).all() and (got[6 + 3] == 0).all()
    Case([40, 1], [6, 70], 4, 2, 64, 16, seed=2, see=see).check()


@pytest.mark.parametrize("d", [64, 128, 80])
def test_tree_attention_nan_stays_where_it_may_be_seen(d):
    """A node whose K or V is not finite reaches the rows that may see it and no other."""
    for what, bad in ((0, float("nan")), (1, float("nan")), (1, float("inf")), (0, float("inf"))):
        c = Case([70], [12], 4, 2, d, 16, seed=d, chain=False)
        node = 5
        clean = c.plain()
        t = 70 + node
        c.pool[c.bt[0, t // 16], c.layer, what, 1, t % 16, 3] = bad
        got, _ = c.run()
        hit = np.zeros((12, 4), bool)
        hit[c.see[0][:, node]] = [False, False, True, True]
        if what == 1:       # only the column of V
            assert not torch.isfinite(got[torch.from_numpy(hit)][:, 3]).any()
            got[:, :, 3] = clean[:, :, 3].float()
        elif np.isnan(bad):
            assert torch.isnan(got[torch.from_numpy(hit)]).all()
            got[torch.from_numpy(hit)] = clean[torch.from_numpy(hit)].float()
        else:               # an infinite key: its score is +-inf by the sign of q
            got[torch.from_numpy(hit)] = clean[torch.from_numpy(hit)].float()
        c.check(got)


@pytest.mark.parametrize("nodes,hq,hkv,d", [(5, 7, 1, 64), (5, 14, 2, 128), (19, 7, 1, 64), (3, 4, 4, 128)])
def test_tree_attention_nan_keys_beside_lanes_without_rows(nodes, hq, hkv, d):
    """Warps of which only some lanes have a query row: their slow path for keys
    that are not finite must not keep the others from the warp's TMEM accesses."""
    g = hq // hkv
    for pos in (3, 66, 70):                     # cached, cached in the tree's tile, the root
        c = Case([70], [nodes], hq, hkv, d, 16, seed=nodes + d)
        clean = c.plain()
        c.pool[c.bt[0, pos // 16], c.layer, 0, hkv - 1, pos % 16, 5] = float("nan")
        got, f = c.run()
        assert f == 0
        sees = torch.tensor([pos < 70 or bool(c.see[0][i][pos - 70]) for i in range(nodes)])
        assert torch.isnan(got[sees][:, hq - g:]).all()
        got[:, hq - g:][sees] = clean[:, hq - g:][sees].float()
        c.check(got)


@pytest.mark.parametrize("k,v", [(1e-6, 1e6), (1e5, 1e-5), (1e12, 1e-12), (1e-20, 1e20)])
def test_tree_attention_value_ranges(k, v):
    Case([100], [9], 8, 2, 128, 16, seed=1, scale=(k, v)).check()
    Case([100], [9], 8, 2, 64, 16, seed=1, scale=(k, v)).check()


def test_tree_attention_mixed_magnitudes_in_one_tile():
    """Values that differ by eight powers of ten from token to token."""
    c = Case([60], [4], 4, 2, 128, 16, seed=8)
    f = 10.0 ** (torch.arange(64) % 9 - 4).double()
    c.kv[0][1] *= f.float()[None, :, None]
    for t in range(64):
        c.pool[c.bt[0, t // 16], c.layer, 1, :, t % 16] = c.kv[0][1][:, t]
    c.check()


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("what", [0, 1])
@pytest.mark.parametrize("factor", [1e4, 1e8, 1e30])
@pytest.mark.parametrize("pre,nodes,big", [(70, 12, [5]), (0, 9, [3, 8]), (100, 90, [7, 40, 41, 80]), (200, 5, [0])])
def test_tree_attention_large_finite_rows_that_nodes_may_not_see(d, what, factor, pre, nodes, big):
    """K or V rows that no node sees, as large as fp32 holds, beside rows that all
    see.  Row by row: a weight is off by 4e-6 of itself and P and V by 2^-22, so
    an output is within 1e-5 of its values' weighted magnitudes."""
    see = [ancestors(p) for p in trees([nodes], np.random.RandomState(d))]
    see[0][:, big] = False
    c = Case([pre], [nodes], 4, 2, d, 16, seed=d + nodes, see=see)
    for b in big:
        t = pre + b
        c.kv[0][what][:, t] *= factor
        c.pool[c.bt[0, t // 16], c.layer, :, :, t % 16] = c.kv[0][:, :, t]
    want = c.plain()
    got, f = c.run()
    assert f == 0
    c.kv[0][1] = c.kv[0][1].abs()
    assert ((got.double() - want).norm(dim=2) <= 1e-5 * c.plain().norm(dim=2)).all()


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("what", [0, 1])
@pytest.mark.parametrize("scale", [1.0, 1e-6, 1e-20])
@pytest.mark.parametrize("pre,nodes,big", [(70, 12, [5]), (0, 9, [3, 8])])
def test_tree_attention_the_types_largest_values_that_nodes_may_not_see(d, what, scale, pre, nodes, big):
    """The same with the largest value that fp32 has, beside V rows of any size."""
    see = [ancestors(p) for p in trees([nodes], np.random.RandomState(d))]
    see[0][:, big] = False
    c = Case([pre], [nodes], 4, 2, d, 16, seed=d + nodes, see=see, scale=(1.0, scale))
    for b in big:
        t = pre + b
        c.kv[0][what][:, t] = torch.finfo(torch.float32).max * c.kv[0][what][:, t].sign()
        c.pool[c.bt[0, t // 16], c.layer, :, :, t % 16] = c.kv[0][:, :, t]
    want = c.plain()
    got, f = c.run()
    assert f == 0
    c.kv[0][1] = c.kv[0][1].abs()
    assert ((got.double() - want).norm(dim=2) <= 1e-5 * c.plain().norm(dim=2)).all()


@pytest.mark.parametrize("d", [64, 128])
def test_tree_attention_large_values_reach_only_their_descendants(d):
    """One node's V is 1e6 times the others': its descendants' outputs are of that
    size, everyone else's are held to their own."""
    c = Case([40], [20], 8, 2, d, 16, seed=d)
    node, t = 4, 44
    c.kv[0][1][:, t] *= 1e6
    c.pool[c.bt[0, t // 16], c.layer, :, :, t % 16] = c.kv[0][:, :, t]
    want = c.plain()
    got, f = c.run()
    assert f == 0
    c.kv[0][1] = c.kv[0][1].abs()
    assert 0 < c.see[0][:, node].sum() < 20
    assert ((got.double() - want).norm(dim=2) <= 1e-5 * c.plain().norm(dim=2)).all()


def test_tree_attention_peaked_scores():
    """Scores of hundreds: nearly every row has one key's weight.  A score of
    500 held to 2^-22 moves a weight by 1.2e-4 where two keys come close."""
    c = Case([90], [5], 4, 2, 128, 16, seed=8)
    c.q *= 60.0
    c.check(rel=2e-4, top_rel=5e-4)


def test_tree_attention_bad_blocks_and_lengths():
    c = Case([40], [4], 4, 2, 64, 16, seed=1)
    good = c.bt.copy()
    for value in (-1, c.pool.shape[0], 1 << 30):
        c.bt = good.copy()
        c.bt[0, 1] = value
        got, f = c.run()
        assert f == BAD_BLOCK
        # the keys of that block read as absent
        k = Case([40], [4], 4, 2, 64, 16, seed=1)
        keep = np.r_[0:16, 32:44]
        k.kv[0] = k.kv[0][:, :, keep]
        k.pre = [24]
        k.check(got)
    c.bt = good[:, :2]
    got, f = c.run()
    assert f & BAD_LENGTH and torch.isfinite(got).all()
    c.bt = good
    c.qs = np.array([0, 5])                     # more nodes than rows of q
    _, f = c.run()
    assert f & BAD_LENGTH


def test_tree_attention_on_another_stream():
    c = Case([300, 20], [8, 8], 8, 2, 128, 16, seed=6)
    want = c.check()
    s = torch.cuda.Stream()
    args = [c.q.cuda(), c.pool.cuda(), c.layer, i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda(), 8, 308]
    torch.cuda.synchronize()
    outs = []
    with torch.cuda.stream(s):
        for _ in range(3):
            outs.append(sp.tree_attention(*args))
    outs += [sp.tree_attention(*args) for _ in range(3)]
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o.cpu(), want)       # the same bits, whatever ran beside it


def test_tree_attention_of_one_cta_between_other_tensor_core_kernels():
    """A call of a single CTA has no second launch: the kernels right before and
    after it in the stream allocate TMEM as it does."""
    from kshipra_b200.quantization import QuantizedLinear
    c = Case([20], [4], 2, 1, 64, 16, seed=3)
    want = c.check().cuda()
    g = torch.Generator().manual_seed(0)
    lin = torch.nn.Linear(256, 256, bias=False)
    lin.weight.data = torch.randn((256, 256), generator=g)
    lin = QuantizedLinear(lin.cuda(), "int8")
    x = torch.randn((64, 256), generator=g).cuda()
    ref = lin(x)
    args = [c.q.cuda(), c.pool.cuda(), c.layer, i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda(), 4, 24]
    got = []
    for _ in range(20):
        got += [(sp.tree_attention(*args), want), (lin(x), ref), (sp.tree_attention(*args), want),
                (sp.tree_attention(*args), want)]
    for a, b in got:
        assert torch.equal(a, b)


def test_tree_attention_offsets_past_32_bits():
    """Blocks whose float offsets lie past 2^31 (and 2^32 bytes past that)."""
    hq, hkv, d, bs, layers = 4, 2, 128, 64, 40
    per = layers * 2 * hkv * bs * d
    nb = (1 << 32) // per + 8
    pool = torch.empty((nb, layers, 2, hkv, bs, d), device="cuda")
    c = Case([150], [6], hq, hkv, d, bs, seed=4, layers=1)
    blocks = [nb - 1, 0, nb // 2 + 3]
    for j, b in enumerate(blocks):
        pool[b, layers - 1] = c.pool[c.bt[0, j], 0].cuda()
    got = sp.tree_attention(c.q.cuda(), pool, layers - 1, i32([blocks]), i32(c.qs), i32(c.pre),
                            c.mask.cuda(), 6, 156)
    c.check(got.cpu())
    # and the move of an accepted node across them
    before = pool[blocks[2], :, :, :, 150 % 64 + 3].clone()
    sp.commit_tree(pool, i32([blocks]), i32([150]), i32([[0, 3]]), i32([2]))
    assert torch.equal(pool[blocks[2], :, :, :, 151 % 64], before)


@pytest.mark.parametrize("seqs,hq,hkv,d,deep,nodes", [
    (130, 6, 2, 64, 200, 5), (700, 4, 2, 64, 90, 3), (700, 2, 1, 128, 90, 3), (24, 16, 2, 64, 900, 30),
    (9, 16, 2, 128, 1900, 40)])
def test_tree_attention_many_items(seqs, hq, hkv, d, deep, nodes):
    """Lines of many items, cut anywhere; sequences without nodes among them."""
    rs = np.random.RandomState(seqs + d)
    pre, lens = rs.randint(0, deep, seqs), rs.randint(0, nodes + 1, seqs)
    lens[seqs // 2] = nodes
    c = Case(pre.tolist(), lens.tolist(), hq, hkv, d, 16, seed=seqs, layers=1)
    c.check()
    assert torch.equal(c.run()[0], c.run()[0])


def test_tree_attention_graph_replay_follows_device_lengths():
    c = Case([200, 90], [8, 8], 8, 2, 64, 16, seed=6)
    args = [c.q.cuda(), c.pool.nan_to_num(0.0).cuda(), c.layer, i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda(), 8, 208]
    out = torch.empty_like(args[0])
    sp.tree_attention(*args, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        sp.tree_attention(*args, out=out)
    args[5].copy_(i32([100, 0]))
    g.replay()
    assert torch.equal(out, sp.tree_attention(*args))


def test_tree_attention_graphs_replayed_side_by_side():
    """Two graphs of one capture stream, replayed on two streams with a larger
    call of the ordinary workspace in between: each has scratch of its own."""
    class Recorder(sp.TreeWorkspace):
        def __init__(self):
            super().__init__()
            self.at = []

        def get(self, nbytes, device):
            buf = super().get(nbytes, device)
            self.at.append(buf.data_ptr())
            return buf

    ws = Recorder()
    cap = torch.cuda.Stream()
    runs = []
    with torch.cuda.stream(cap):
        for d, seed in ((64, 6), (128, 7), (64, 8)):
            c = Case([900, 300], [8, 8], 8, 2, d, 16, seed=seed)
            args = [c.q.cuda(), c.pool.cuda(), c.layer, i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda(), 8, 908]
            want = sp.tree_attention(*args, ws=ws)
            out = torch.zeros_like(want)
            cap.synchronize()
            c.check(want.cpu())
            runs.append((args, out, want, torch.cuda.CUDAGraph()))
        for args, out, _, graph in runs:
            with torch.cuda.graph(graph, stream=cap):
                sp.tree_attention(*args, out=out, ws=ws)
                sp.tree_attention(*args, out=out, ws=ws)
        after = sp.tree_attention(*runs[1][0], ws=ws)
    torch.cuda.synchronize()
    eager, held = ws.at[:3] + ws.at[-1:], [set(ws.at[3 + 2 * i:5 + 2 * i]) for i in range(3)]
    assert len(set(eager)) == 1 and torch.equal(after, runs[1][2])
    assert not (held[0] & held[1] or held[0] & held[2] or held[1] & held[2] or set(eager) & set.union(*held))
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(30):
        for stream, (_, _, _, graph) in zip(streams, runs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in runs:
        assert torch.equal(out, want)


# --------------------------------------------------------------------------- #
# probabilities
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("vocab", [1, 3, 31, 1024, 1027, 32003, 151936])
def test_target_probs(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn((7, vocab), generator=g) * 6
    x[1] -= 300.0
    x[2, vocab // 2:] = float("-inf") if vocab > 1 else 0.0
    x[3] = x[3].round()                          # ties
    t = torch.tensor([1.0, 0.7, 2.0, 0.0, 0.5, 0.0, 100.0])
    x[5] = 2.5                                   # every entry is the maximum
    xd = x.cuda()
    got = sp.target_probs(xd, t.cuda()).cpu().double()
    for r in range(7):
        if t[r] > 0:
            want = torch.softmax((x[r].double() - x[r].max().double()) / t[r].double(), 0)
            assert ((got[r] - want).abs() <= 1e-5 * want + 1e-37).all(), r
        else:
            assert got[r].nonzero().view(-1).tolist() == [int(x[r].argmax())] and got[r].max() == 1
    assert torch.equal(sp.target_probs(xd), sp.target_probs(xd, torch.ones(7, device="cuda")))
    # rows of a wider buffer, into another, and in place
    wide = torch.full((7, vocab + 5), float("nan"), device="cuda")
    wide[:, 2:2 + vocab] = xd
    dst = torch.full((7, vocab + 3), -1.0, device="cuda")
    sp.target_probs(wide[:, 2:2 + vocab], t.cuda(), out=dst[:, 1:1 + vocab])
    assert torch.equal(dst[:, 1:1 + vocab].cpu().double(), got)
    assert (dst[:, 0] == -1).all() and (dst[:, 1 + vocab:] == -1).all()
    assert torch.equal(sp.target_probs(xd, t.cuda(), out=xd).cpu().double(), got)


@pytest.mark.parametrize("m,vocab", [(601, 1000), (1300, 3), (2400, 6), (600, 20483), (151, 39998), (83, 151936)])
def test_target_probs_many_rows(m, vocab):
    """Rows on 16-byte boundaries and not give the same bits, however many."""
    g = torch.Generator().manual_seed(m)
    width = (vocab + 3) // 4 * 4 + 4
    x = (torch.randn((m, width), generator=g) * 5).cuda()
    x[3, :vocab] = float("-inf")
    x[4, vocab // 2] = float("nan")
    x[5, :vocab // 2] = float("-inf")
    t = (torch.rand(m, generator=g) + 0.5).cuda()
    t[::7] = 0.0
    out = torch.full_like(x, -1.0)
    sp.target_probs(x[:, :vocab], t, out=out[:, :vocab])
    assert (out[:, vocab:] == -1).all()
    off = torch.empty((m, width + 1), device="cuda")
    off[:, 1:1 + vocab] = x[:, :vocab]
    want = sp.target_probs(off[:, 1:1 + vocab], t)
    assert torch.equal(out[:, :vocab].nan_to_num(7.0), want.nan_to_num(7.0))
    for r in (0, 1, 2, 5, 14, m - 2, m - 1):
        row = x[r, :vocab].cpu().double()
        if float(t[r]) > 0:
            ref = torch.softmax((row - row.max()) / t[r].cpu().double(), 0)
            assert ((out[r, :vocab].cpu().double() - ref).abs() <= 1e-5 * ref + 1e-37).all(), r
        else:
            assert out[r, :vocab].nonzero().view(-1).tolist() == [int(row.argmax())]
    assert torch.isnan(out[3, :vocab]).all() and torch.isnan(out[4, :vocab]).all()
    same = x.clone()
    sp.target_probs(same[:, :vocab], t, out=same[:, :vocab])
    assert torch.equal(same[:, :vocab].nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("vocab", [8, 5000, 151936, 420001])
def test_target_probs_greedy_ties_of_signed_zeros(vocab):
    """-0 and +0 are one value: the first of them is the maximum."""
    x = torch.full((3, vocab), -1.0)
    x[0, 2], x[0, vocab - 2] = -0.0, 0.0
    x[1, 3], x[1, vocab - 3] = 0.0, -0.0
    x[2] = -0.0
    got = sp.target_probs(x.cuda(), torch.zeros(3, device="cuda")).cpu()
    assert [r.nonzero().view(-1).tolist() for r in got] == [[2], [3], [0]] and got.max() == 1


@pytest.mark.parametrize("vocab", [8, 5000, 151936, 420001])
def test_target_probs_greedy_rows_with_nan(vocab):
    """NaN is the largest, as torch.argmax and the batch lm_head take it; its sign
    does not matter."""
    x = torch.randn((4, vocab), generator=torch.Generator().manual_seed(vocab))
    x[0, vocab - 2] = float("nan")
    x[0, 1] = float("inf")
    x[1, 3] = x[1, 5] = float("nan")
    x[2] = float("nan")
    x.view(torch.int32)[3, 4] = -1
    got = sp.target_probs(x.cuda(), torch.zeros(4, device="cuda")).cpu()
    assert [r.nonzero().view(-1).tolist() for r in got] == [[vocab - 2], [3], [0], [4]] and got.max() == 1


@pytest.mark.parametrize("vocab", [7, 5000, 420001])
def test_target_probs_at_the_smallest_temperatures(vocab):
    """1 / T overflows below 2^-127: what is left is the softmax's limit, all on the
    maxima alike."""
    x = torch.randn((4, vocab), generator=torch.Generator().manual_seed(vocab))
    x[:, 2] = x[:, 5] = 9.0
    x[1, 5] = 9.0 - 1e-6                        # the next fp32 below 9
    x[2, 3] = float("-inf")
    t = torch.tensor([1e-40, 1e-45, 3e-39, 1e-38])
    assert (t > 0).all()
    got = sp.target_probs(x.cuda(), t.cuda()).cpu()
    want = torch.zeros_like(got)
    want[:, 2] = want[:, 5] = 0.5
    want[1, 2], want[1, 5] = 1.0, 0.0
    assert torch.equal(got, want)
    assert torch.isnan(sp.target_probs(x[:1].cuda(), torch.full((1,), float("nan"), device="cuda"))).all()


def test_target_probs_rows_past_a_clusters_shared_memory():
    """Rows that are read three times; also in place and from odd addresses."""
    vocab = 500009
    x = torch.randn((3, vocab + 3), generator=torch.Generator().manual_seed(1)) * 5
    t = torch.tensor([0.7, 0.0, 1.3])
    xd = x.cuda()[:, 1:1 + vocab]
    got = sp.target_probs(xd, t.cuda())
    for r in (0, 2):
        want = torch.softmax(x[r, 1:1 + vocab].double() / t[r].double(), 0)
        assert ((got[r].cpu().double() - want).abs() <= 1e-5 * want + 1e-37).all()
    assert got[1].nonzero().view(-1).tolist() == [int(x[1, 1:1 + vocab].argmax())]
    assert torch.equal(sp.target_probs(xd, t.cuda(), out=xd), got)


@pytest.mark.parametrize("vocab", [151936, 409600, 409601, 3000001])
def test_target_probs_of_flat_rows(vocab):
    """Terms of one size: the sum of hundreds of thousands is good to 1e-6 and a term
    to 2e-6 (2 ulp, arguments below 1)."""
    x = torch.randn((3, vocab), generator=torch.Generator().manual_seed(vocab))
    t = torch.tensor([50.0, 20.0, 1000.0, 3.0, 1.0, 7.0])
    x = torch.cat([x, torch.full((3, vocab), -1.0)])        # equal terms round the same way at each addition
    x[3:, 5] = 0.0
    want = torch.softmax(x.double() / t[:, None].double(), 1)
    got = sp.target_probs(x.cuda(), t.cuda()).cpu().double()
    assert ((got - want).abs() <= 3e-6 * want).all()


def test_target_probs_not_finite_rows():
    x = torch.zeros((4, 200))
    x[0, 5] = float("nan")
    x[1] = float("-inf")
    x[2, 7] = float("inf")
    got = sp.target_probs(x.cuda()).cpu()
    assert torch.isnan(got[0]).all() and torch.isnan(got[1]).all() and torch.isnan(got[2, 7])
    assert torch.allclose(got[3], torch.full((200,), 1 / 200))
    assert sp.target_probs(x.cuda()[:0]).shape == (0, 200)


# --------------------------------------------------------------------------- #
# verification
# --------------------------------------------------------------------------- #

def plain_verify(tok, par, P, Q, greedy, u, us):
    """One sequence, in 64 bits."""
    n, cur, took = len(tok), 0, [0]
    if greedy is not None:
        for i in range(1, n):
            if par[i] == cur and tok[i] == greedy[cur]:
                cur = i
                took.append(i)
        return took, greedy[cur]
    r, z = P[0].copy(), 1.0
    for i in range(1, n):
        if par[i] != cur:
            continue
        q = 1.0 if Q is None else Q[cur][tok[i]]
        if u[i] * z * q < r[tok[i]]:
            cur, z, r = i, 1.0, P[i].copy()
            took.append(i)
        elif Q is None:
            z -= r[tok[i]]
            r[tok[i]] = 0.0
        else:
            r = np.maximum(r - z * Q[cur], 0.0)
            z = r.sum()
    if not r.sum() > 0:
        r = P[cur]
    c = np.cumsum(r)
    return took, int(np.argmax(c > us * c[-1]))


def random_batch(lens, vocab, kind, seed, chain=False):
    rs = np.random.RandomState(seed)
    par = trees(lens, rs, chain)
    T = sum(lens)
    x = rs.randn(T, vocab) * 2.0
    P = np.exp(x - x.max(1, keepdims=True))
    P = (P / P.sum(1, keepdims=True)).astype(np.float32)
    y = x + 0.8 * rs.randn(T, vocab)
    Q = np.exp(y - y.max(1, keepdims=True))
    Q = (Q / Q.sum(1, keepdims=True)).astype(np.float32)
    tok = np.zeros(T, np.int64)
    at = 0
    for n, p in zip(lens, par):
        for i in range(1, n):
            row = at + max(int(p[i]), 0)
            tok[at + i] = (rs.choice(vocab, p=Q[row].astype(np.float64) / Q[row].sum(dtype=np.float64))
                           if kind == "drawn" else Q[row].argsort()[-1 - rs.randint(min(3, vocab))])
        at += n
    u, us = rs.rand(T).astype(np.float32), rs.rand(len(lens)).astype(np.float32)
    return tok, par, P, Q, u, us


def check_verify(lens, vocab, kind, seed, chain=False, wide=0):
    tok, par, P, Q, u, us = random_batch(lens, vocab, kind, seed, chain)
    qs = np.concatenate([[0], np.cumsum(lens)])
    greedy = P.argmax(1) if kind == "greedy" else None

    def rows(a):
        t = torch.full((a.shape[0], vocab + wide), float("nan"), device="cuda")
        t[:, wide // 2:wide // 2 + vocab] = torch.from_numpy(a).cuda()
        return t[:, wide // 2:wide // 2 + vocab] if wide else t.contiguous()

    kw = {}
    if kind == "greedy":
        kw["target_tokens"] = torch.from_numpy(greedy).cuda()
    else:
        kw.update(target_probs=rows(P), u_accept=torch.from_numpy(u).cuda(),
                  u_sample=torch.from_numpy(us).cuda())
        if kind == "drawn":
            kw["draft_probs"] = rows(Q)
    flags = new_flags()
    most = max(max(lens), 1)
    path, ln, nxt = sp.verify_tree(torch.from_numpy(tok).cuda(), i32(np.concatenate(par)), i32(qs),
                                   most, flags=flags, **kw)
    assert int(flags) == 0
    P64, Q64 = P.astype(np.float64), Q.astype(np.float64)
    for s, n in enumerate(lens):
        a, e = qs[s], qs[s + 1]
        row = path[s].tolist()
        if n == 0:
            assert row == [-1] * most and int(ln[s]) == 0 and int(nxt[s]) == -1
            continue
        took, t = plain_verify(tok[a:e], par[s], P64[a:e], Q64[a:e] if kind == "drawn" else None,
                               None if greedy is None else greedy[a:e], u[a:e].astype(np.float64),
                               float(us[s]))
        assert row == took + [-1] * (most - len(took)), (s, row, took)
        assert int(ln[s]) == len(took) and int(nxt[s]) == t, (s, int(nxt[s]), t)


@pytest.mark.parametrize("kind", ["drawn", "fixed", "greedy"])
@pytest.mark.parametrize("vocab", [2, 37, 1000, 5003])
@pytest.mark.parametrize("lens", [[1], [2], [5, 0, 9], [30] * 20])
def test_verify_tree(kind, vocab, lens):
    check_verify(lens, vocab, kind, seed=vocab + len(lens))
    check_verify(lens, vocab, kind, seed=vocab + len(lens) + 1, chain=True)


@pytest.mark.parametrize("kind", ["drawn", "fixed"])
def test_verify_tree_large_vocabularies_and_row_strides(kind):
    check_verify([7, 3], 50257, kind, seed=1)
    check_verify([6], 151936, kind, seed=2)
    check_verify([9, 4, 1], 4001, kind, seed=3, wide=6)
    check_verify([200, 256], 64, kind, seed=4)


@pytest.mark.parametrize("kind", ["drawn", "fixed"])
def test_verify_tree_many_sequences_over_a_large_vocabulary(kind):
    """So many sequences that each has one CTA, whose warps' pieces hold more steps
    than there are slots for their sums."""
    S, V = 300, 131073
    g = torch.Generator(device="cuda").manual_seed(5)
    P = torch.softmax(torch.randn((2 * S, V), generator=g, device="cuda") * 3, 1)
    Q = torch.softmax(torch.randn((2 * S, V), generator=g, device="cuda") * 3, 1)
    tok = torch.multinomial(Q, 1, generator=g).view(-1)
    tok[1::2] = torch.where(torch.arange(S, device="cuda") % 2 == 0, P[::2].argmax(1), tok[::2])
    u, us = torch.rand(2 * S, generator=g, device="cuda"), torch.rand(S, generator=g, device="cuda")
    us[:3] = torch.tensor([0.0, 0.9999999, 0.5], device="cuda")
    path, ln, nxt = sp.verify_tree(tok, i32([-1, 0] * S), i32(np.arange(S + 1) * 2), 2, target_probs=P,
                                   draft_probs=Q if kind == "drawn" else None, u_accept=u, u_sample=us)
    for s in range(S):
        p, t = P[2 * s].double(), int(tok[2 * s + 1])
        q = Q[2 * s].double() if kind == "drawn" else None
        if float(u[2 * s + 1].double() * (1.0 if q is None else q[t])) < float(p[t]):
            want, p = [0, 1], P[2 * s + 1].double()
        else:
            want = [0, -1]
            if q is None:
                p[t] = 0.0
            else:
                p = (p - q).clamp(min=0)
        c = p.cumsum(0)
        assert path[s].tolist() == want and int(ln[s]) == 2 + min(want[1], 0)
        assert int(nxt[s]) == int((c > us[s].double() * c[-1]).to(torch.int8).argmax()), s
    assert 0 < int((ln == 2).sum()) < S           # both ends were walked


@pytest.mark.parametrize("kind", ["drawn", "fixed"])
def test_verified_tokens_follow_the_target(kind):
    """The first emitted token's distribution is the target's, whatever was
    drafted: counts over 40000 sequences against P, chi-square with 7 degrees
    of freedom below 40 (exceeded with probability 1e-6; the seed is fixed)."""
    S, V = 40000, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    P0 = torch.softmax(torch.randn(V, generator=g, device="cuda") * 1.2, 0)
    Q0 = torch.softmax(torch.randn(V, generator=g, device="cuda") * 1.2, 0)
    par = [-1, 0, 0, 0]
    P, Q = P0.expand(4 * S, V).contiguous(), Q0.expand(4 * S, V).contiguous()
    if kind == "drawn":
        tok = torch.multinomial(Q0, 4 * S, replacement=True, generator=g)
    else:
        tok = Q0.topk(4).indices.repeat(S)
    path, ln, nxt = sp.verify_tree(
        tok, i32(par * S), i32(np.arange(S + 1) * 4), 4, target_probs=P,
        draft_probs=Q if kind == "drawn" else None,
        u_accept=torch.rand(4 * S, generator=g, device="cuda"),
        u_sample=torch.rand(S, generator=g, device="cuda"))
    first = torch.where(ln > 1, tok.view(S, 4).gather(1, path[:, 1:2].clamp(min=0).long()).view(-1), nxt)
    count = torch.bincount(first, minlength=V).double().cpu()
    want = P0.double().cpu() * S
    assert float(((count - want) ** 2 / want).sum()) < 40.0


def test_verify_tree_edges():
    V = 100
    P = torch.zeros((3, V), device="cuda")
    P[0, 7] = 1.0
    P[1, 9], P[2, 11] = 1.0, 1.0
    tok = torch.tensor([0, 7, 9], device="cuda")
    one = lambda x: torch.full((1,), x, device="cuda")  # noqa: E731
    u = torch.zeros(3, device="cuda")
    # point masses: accepted to the end, the last row's token
    path, ln, nxt = sp.verify_tree(tok, i32([-1, 0, 1]), i32([0, 3]), 3, target_probs=P, u_accept=u,
                                   u_sample=one(0.999))
    assert path.tolist() == [[0, 1, 2]] and ln.item() == 3 and nxt.item() == 11
    # P == Q: a refusal would leave nothing, the node's own row stands in
    path, ln, nxt = sp.verify_tree(tok, i32([-1, 0, 1]), i32([0, 3]), 3, target_probs=P,
                                   draft_probs=P, u_accept=torch.ones(3, device="cuda"),
                                   u_sample=one(0.5))
    assert ln.item() == 1 and nxt.item() == 7
    # a token outside the vocabulary is never accepted; a later parent is no parent
    for t, par, bit in ((torch.tensor([0, V, 9], device="cuda"), [-1, 0, 0], BAD_TOKEN),
                        (torch.tensor([0, -1, 9], device="cuda"), [-1, 0, 0], BAD_TOKEN),
                        (tok, [-1, 2, 1], BAD_PARENT)):
        flags = new_flags()
        _, ln, nxt = sp.verify_tree(t, i32(par), i32([0, 3]), 3, target_probs=P, u_accept=u,
                                    u_sample=one(0.5), flags=flags)
        assert ln.item() == 1 and nxt.item() == 7 and int(flags) == bit
    # a row without mass, or with NaN
    for bad in (0.0, float("nan")):
        flags = new_flags()
        _, ln, nxt = sp.verify_tree(tok[:1], i32([-1]), i32([0, 1]), 1, flags=flags, u_sample=one(0.5),
                                    target_probs=torch.full((1, V), bad, device="cuda"), u_accept=u[:1])
        assert int(flags) == BAD_PROBS and ln.item() == 1 and nxt.item() == 0
    # q_start past the rows
    flags = new_flags()
    path, ln, nxt = sp.verify_tree(tok, i32([-1, 0, 1]), i32([0, 4]), 4, target_tokens=tok, flags=flags)
    assert int(flags) == BAD_LENGTH and ln.item() == 0 and nxt.item() == -1


# --------------------------------------------------------------------------- #
# commit
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("hkv,d,block,layers", [(2, 64, 16, 3), (8, 128, 16, 3), (1, 6, 7, 3), (3, 5, 1, 3),
                                                (2, 24, 16, 260), (2, 6, 16, 260)])
def test_commit_tree(hkv, d, block, layers):
    rs = np.random.RandomState(d)
    lens = [8, 1, 40, 5, 0]
    pre = [13, 0, 50, 16, 4]
    need = [max(1, -(-(p + n) // block)) for p, n in zip(pre, lens)]
    nb = sum(need) + 1
    order = rs.permutation(nb)
    bt = np.zeros((5, max(need)), np.int64)
    at = 0
    for s in range(5):
        bt[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
    path = np.full((5, 40), -1)
    for s, p in enumerate([[0, 2, 3, 7], [0], list(range(0, 40, 2)), [0, 1, 2], []]):
        path[s, :len(p)] = p
    ln = (path >= 0).sum(1)
    pool = torch.from_numpy(rs.randn(nb, layers, 2, hkv, block, d).astype(np.float32))
    want = pool.clone()
    for s in range(5):
        for j in range(ln[s]):
            x, y = pre[s] + path[s, j], pre[s] + j
            want[bt[s, y // block], :, :, :, y % block] = want[bt[s, x // block], :, :, :, x % block].clone()
    dev, flags = pool.cuda(), new_flags()
    got = sp.commit_tree(dev, i32(bt), i32(pre), i32(path), i32(ln), flags=flags)
    assert int(flags) == 0 and got.tolist() == [p + n for p, n in zip(pre, ln)]
    assert torch.equal(dev.cpu(), want)


def test_commit_tree_reports_bad_paths():
    pool = torch.randn(4, 2, 2, 2, 16, 64, device="cuda")
    before = pool.clone()
    for path, ln, bt, bit in (([[0, 3, 2]], [3], [[0, 1]], BAD_LENGTH), ([[0, -1, 2]], [3], [[0, 1]], BAD_LENGTH),
                              ([[0, 2]], [5], [[0, 1]], BAD_LENGTH), ([[0, 2]], [-1], [[0, 1]], BAD_LENGTH),
                              ([[0, 20]], [2], [[0, 9]], BAD_BLOCK), ([[0, 40]], [2], [[0, 1]], BAD_BLOCK)):
        flags = new_flags()
        sp.commit_tree(pool, i32(bt), i32([2]), i32(path), i32(ln), flags=flags)
        assert int(flags) == bit, (path, ln)
    # 3 -> 1 of the first path was good, everything else stayed
    before[0, :, :, :, 3] = before[0, :, :, :, 5]
    assert torch.equal(pool, before)


# --------------------------------------------------------------------------- #
# refusals and the decoder
# --------------------------------------------------------------------------- #

def test_refusals():
    c = Case([10], [4], 4, 2, 64, 16)
    q, pool, bt, qs, pre, mask = c.q.cuda(), c.pool.cuda(), i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda()
    with pytest.raises(_lib.KshipraLibraryError):
        sp.tree_attention(c.q, pool, 0, bt, qs, pre, mask, 4, 14)
    for bad in (lambda: sp.tree_attention(q.half(), pool, 0, bt, qs, pre, mask, 4, 14),
                lambda: sp.tree_attention(q.transpose(0, 1), pool, 0, bt, qs, pre, mask, 4, 14),
                lambda: sp.tree_attention(q[:, :3].contiguous(), pool, 0, bt, qs, pre, mask, 4, 14),
                lambda: sp.tree_attention(q, pool, 2, bt, qs, pre, mask, 4, 14),
                lambda: sp.tree_attention(q, pool, 0, bt.long(), qs, pre, mask, 4, 14),
                lambda: sp.tree_attention(q, pool, 0, bt, qs[:1], pre, mask, 4, 14),
                lambda: sp.tree_attention(q, pool, 0, bt, qs, pre, mask[:2], 4, 14),
                lambda: sp.tree_attention(q, pool, 0, bt, qs, pre, mask, 257, 270),
                lambda: sp.tree_attention(q, pool, 0, bt, qs, pre, mask, 4, 14, out=q[:2]),
                lambda: sp.tree_tables(pre, pre, 10, 16, 4, 1),
                lambda: sp.tree_tables(pre, pre, 10, 16, 4, 9, block_tables=bt),
                lambda: sp.tree_tables(pre, pre, 10, 16, 300, 1, block_tables=bt, parents=i32([0] * 10)),
                lambda: sp.tree_tables(pre, pre, 10, 16, 4, 1, block_tables=bt, parents=i32([0])),
                lambda: sp.target_probs(q[0].t()),
                lambda: sp.target_probs(q[0], torch.ones(2, device="cuda")),
                lambda: sp.verify_tree(qs.long(), qs, qs, 2),
                lambda: sp.verify_tree(qs.long(), qs, qs, 2, target_tokens=qs),
                lambda: sp.verify_tree(qs.long(), qs, qs, 2, target_probs=q[0][:2].contiguous()),
                lambda: sp.commit_tree(pool, bt, pre, qs, pre),
                lambda: sp.commit_tree(pool.double(), bt, pre, bt, pre)):
        with pytest.raises(ValueError):
            bad()


def test_status_words_are_checked_before_the_launch():
    c = Case([10], [4], 4, 2, 64, 16)
    q, pool, bt, qs, pre, mask = c.q.cuda(), c.pool.cuda(), i32(c.bt), i32(c.qs), i32(c.pre), c.mask.cuda()
    par, tok = i32([-1, 0, 0, 1]), torch.zeros(4, dtype=torch.int64, device="cuda")
    path, ln = sp.verify_tree(tok, par, qs, 4, target_tokens=tok)[:2]
    calls = (lambda f: sp.tree_tables(pre, i32([4]), 4, 16, 4, bt.shape[1], block_tables=bt, parents=par, flags=f),
             lambda f: sp.tree_attention(q, pool, 0, bt, qs, pre, mask, 4, 14, flags=f),
             lambda f: sp.verify_tree(tok, par, qs, 4, target_tokens=tok, flags=f),
             lambda f: sp.commit_tree(pool, bt, pre, path, ln, flags=f))
    for call in calls:
        call(new_flags())
        with pytest.raises(_lib.KshipraLibraryError):
            call(torch.zeros(1, dtype=torch.int32))
        with pytest.raises(ValueError):
            call(torch.zeros(1, dtype=torch.int64, device="cuda"))


@pytest.fixture(scope="module")
def tiny():
    from kshipra_b200.config import TINY_LLAMA
    from kshipra_b200.model import KshipraModel
    from kshipra_b200.weights import synthetic_state_dict
    sd = synthetic_state_dict(TINY_LLAMA, seed=0)
    return KshipraModel(config=TINY_LLAMA, state_dict=sd, quantize="int8", device=torch.device("cuda", 0))


def prompts_of(vocab):
    rs = np.random.RandomState(7)
    a = rs.randint(0, vocab, 12).tolist()
    return [a * 3, rs.randint(0, vocab, 29).tolist(), a + a[:5], [5]]


class Oracle:
    """Drafts the known continuation with wrong branches beside it."""

    max_nodes = 12

    def __init__(self, streams, vocab):
        self.streams, self.vocab = streams, vocab

    def propose(self, tokens):
        full = next(s for s in self.streams if s[:len(tokens)] == list(tokens))
        toks, par, at = [tokens[-1]], [-1], 0
        for t in full[len(tokens):len(tokens) + 4]:
            toks += [(t + 1) % self.vocab, t]
            par += [at, at]
            at = len(toks) - 1
        return toks, par


def test_decoder_greedy_stream_is_generates(tiny):
    prompts = prompts_of(tiny.vocab_size)
    want = [tiny.generate(p, max_new_tokens=20, block_size=16) for p in prompts]
    dec = sp.SpeculativeDecoder(tiny, block_size=16)
    assert dec.generate(prompts, max_new_tokens=20) == want
    # drafts that come true are kept: four tokens and the one after them a step
    dec = sp.SpeculativeDecoder(tiny, Oracle([p + w for p, w in zip(prompts, want)], tiny.vocab_size),
                                block_size=24)
    assert dec.generate(prompts, max_new_tokens=20) == want
    assert dec.emitted == 80 and dec.steps == 4
    eos = want[0][4]
    cut = [w[:w.index(eos) + 1] if eos in w else w for w in want]
    assert sp.SpeculativeDecoder(tiny).generate(prompts, 20, eos_token_id=eos) == cut


def test_decoder_drafts_only_what_can_be_emitted(tiny, monkeypatch):
    """A prompt that repeats itself up to the end of the position table: generate
    feeds the table's last position, and no draft lies behind it."""
    a = np.random.RandomState(7).randint(0, tiny.vocab_size, 12).tolist()
    prompts = [(a * 200)[:tiny.max_positions - 8], a * 3, a]
    want = [tiny.generate(p, 9, block_size=16) for p in prompts]
    last = []
    real = sp.tree_tables

    def spy(prefix, new, *args, **kw):
        out = real(prefix, new, *args, **kw)
        last.extend((out[2][out[0][1:].long() - 1]).tolist())
        last.append(int(out[2].max()))
        return out

    monkeypatch.setattr(sp, "tree_tables", spy)
    assert sp.SpeculativeDecoder(tiny).generate(prompts, 9) == want
    assert max(last) == tiny.max_positions - 1
    last.clear()
    drafts = Oracle([p + w for p, w in zip(prompts, want)], tiny.vocab_size)
    assert sp.SpeculativeDecoder(tiny, drafts).generate(prompts[:1], 9) == want[:1]
    assert max(last) == tiny.max_positions - 1
    # the model's own limit still holds, as it does for generate
    from kshipra_b200.model import KshipraDeviceError
    for run in (tiny.generate, lambda p, n: sp.SpeculativeDecoder(tiny).generate([p], n)):
        with pytest.raises(KshipraDeviceError):
            run(prompts[0], 12)


def test_decoder_counts_the_tokens_that_it_returns(tiny):
    """An end token amid accepted drafts: what comes after it is not emitted."""
    prompts = prompts_of(tiny.vocab_size)
    want = [tiny.generate(p, max_new_tokens=20, block_size=16) for p in prompts]
    drafts = Oracle([p + w for p, w in zip(prompts, want)], tiny.vocab_size)
    for eos in {w[2] for w in want} | {w[7] for w in want}:
        cut = [w[:w.index(eos) + 1] if eos in w else w for w in want]
        dec = sp.SpeculativeDecoder(tiny, drafts)
        assert dec.generate(prompts, 20, eos_token_id=eos) == cut
        assert dec.emitted == sum(len(w) for w in cut)


def test_decoder_reports_what_the_prefill_found(tiny):
    """A prompt token outside the vocabulary, also where no step follows."""
    from kshipra_b200.model import KshipraDeviceError
    for n in (1, 4):
        for dec in (sp.SpeculativeDecoder(tiny), sp.SpeculativeDecoder(tiny, temperature=0.7)):
            with pytest.raises(KshipraDeviceError):
                dec.generate([[1, 2], [tiny.vocab_size + 5, 3]], n)
            assert int(tiny.flags) == 0


def test_decoder_refuses_trees_past_the_proposers_limit(tiny):
    class Many:
        max_nodes = 2

        def propose(self, tokens):
            return [tokens[-1], 1, 2, 3], [-1, 0, 1, 2]

    with pytest.raises(ValueError):
        sp.SpeculativeDecoder(tiny, Many()).generate([[1, 2, 3]], 9)


def test_decoder_sampling(tiny):
    """Temperature: the stream is the generator's, and a tiny temperature is greedy."""
    prompts = prompts_of(tiny.vocab_size)
    runs = [sp.SpeculativeDecoder(tiny, temperature=0.8, generator=torch.Generator("cuda").manual_seed(k))
            .generate(prompts, 12) for k in (1, 1, 2)]
    assert runs[0] == runs[1] != runs[2]
    assert all(len(r) == 12 and all(0 <= t < tiny.vocab_size for t in r) for r in runs[0])
    cold = sp.SpeculativeDecoder(tiny, temperature=1e-4, generator=torch.Generator("cuda").manual_seed(1))
    assert cold.generate(prompts, 12) == [tiny.generate(p, 12, block_size=16) for p in prompts]
