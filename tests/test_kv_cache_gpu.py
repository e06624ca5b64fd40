"""The 16-bit paged cache on the GPU against plain implementations in 64 bits.

Tolerances.  Attention: the framework's bound for its fp32 attention, a relative
L2 error of 1e-5 against 64 bits on the same (already rounded) K and V; single
elements within 8e-5 of the largest value the row can reach (scores of size 16
held to 2^-22 relative move a probability by 16 * 2^-22 = 4e-6, a probability of
two bf16 terms is held to 2^-18 = 4e-6, and an output is a mean of values with
such weights; the factor 10 is for rows of few keys).  Written rows: without norms the
fp32 result is rounded like torch's, bit by bit; with norms, the fp32 sums and
products err by at most 16 * 2^-24 of |y1| + |y2| (a sum of squares in a tree of
at most 12 steps, half of that after the root, a root, a quotient, four
products, a sum), and a stored value by half a step of its type beside that.
Pages are exact.
"""

import threading

import numpy as np
import pytest
import torch

from kshipra_b200 import _lib
from kshipra_b200 import kv_cache as kv
from kshipra_b200.chunked_prefill import paged_attention

pytestmark = pytest.mark.gpu

BAD_BLOCK, BAD_SLOT, BAD_POSITION, BAD_LENGTH, BAD_PARENT, NO_PAGE = 2, 4, 8, 32, 128, 512
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def i64(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int64).cuda()


def new_flags():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


# --------------------------------------------------------------------------- #
# attention
# --------------------------------------------------------------------------- #

class Batch:
    """Sequences (cached, new) over a shuffled pool."""

    def __init__(self, seqs, heads, kv_heads, d, block, dtype, layers=1, seed=0, spare=3, first_row=0, tail_rows=0,
                 q_scale=2.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rs = np.random.RandomState(seed)
        self.pre, self.new = [p for p, _ in seqs], [n for _, n in seqs]
        need = [max(1, -(-(p + n) // block)) for p, n in seqs]
        nb = sum(need) + spare
        ids = rs.permutation(nb)
        table, at = np.zeros((len(seqs), max(need)), np.int64), 0
        for i, n in enumerate(need):
            table[i, :n] = ids[at:at + n]
            at += n
        self.unused = ids[at:]
        qs = first_row + np.concatenate([[0], np.cumsum(self.new)])
        self.total = int(qs[-1]) + tail_rows
        self.table, self.q_start, self.prefix = i32(table), i32(qs), i32(self.pre)
        self.qs = qs
        self.pool = torch.randn(nb, layers, 2, kv_heads, block, d, generator=g, device="cuda").to(dtype)
        self.q = torch.randn(max(self.total, 1), heads, d, generator=g, device="cuda") * q_scale
        self.layer = layers - 1
        self.block, self.g = block, heads // kv_heads
        self.max_q, self.max_total = max(self.new), max(p + n for p, n in seqs)

    def run(self, **kw):
        return kv.cache_attention(self.q, self.pool, self.layer, self.table, self.q_start, self.prefix, self.max_q,
                                  self.max_total, **kw)

    def seq(self, s):
        """K and V [2, Hkv, length, D] of a sequence in 64 bits."""
        ln = self.pre[s] + self.new[s]
        used = self.table[s, : -(-ln // self.block)].long()
        x = self.pool[used, self.layer].permute(1, 2, 0, 3, 4)
        return x.reshape(2, x.shape[1], -1, x.shape[-1])[:, :, :ln].double()

    def want(self):
        out = torch.full(self.q.shape, float("nan"), dtype=torch.float64, device="cuda")
        for s, (p, n) in enumerate(zip(self.pre, self.new)):
            if n == 0:
                continue
            k, v = self.seq(s).repeat_interleave(self.g, 1)
            a = int(self.qs[s])
            x = torch.einsum("nhd,hkd->hnk", self.q[a:a + n].double(), k) / self.q.shape[2] ** 0.5
            hide = torch.ones(n, p + n, dtype=torch.bool, device="cuda").triu(p + 1)
            w = torch.softmax(x.masked_fill(hide, float("-inf")), -1)
            out[a:a + n] = torch.einsum("hnk,hkd->nhd", w, v)
        return out

    def check(self, got, want=None):
        want = self.want() if want is None else want
        on = ~torch.isnan(want)
        assert torch.isfinite(got[on]).all()
        diff = (got.double() - want)[on]
        if on.any():
            assert float(diff.norm()) <= 1e-5 * float(want[on].norm())
            top = max(float(torch.nan_to_num(self.seq(s)[1].abs(), nan=0.0, posinf=0.0).max())
                      for s in range(len(self.new)) if self.new[s])
            assert float(diff.abs().max()) <= 8e-5 * top


LENGTHS = [
    [(0, 1)],
    [(540, 1)],
    [(0, 5), (3, 1), (127, 1), (128, 1), (126, 1), (255, 2), (64, 64), (63, 1)],
    [(0, 300)],
    [(200, 129), (0, 0), (1000, 1), (5, 37), (0, 128), (31, 0), (129, 255)],
    [(5000, 1), (4999, 3), (17, 1), (2, 1)],
]
SHAPES = [(14, 2, 64), (32, 8, 128), (4, 4, 64), (3, 1, 128), (16, 1, 128), (6, 2, 64)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", range(len(LENGTHS)))
def test_attention(lengths, shape, dtype):
    b = Batch(LENGTHS[lengths], *shape, 16, dtype, layers=2, seed=lengths)
    f = new_flags()
    b.check(b.run(flags=f))
    assert int(f) == 0


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("block", [1, 2, 7, 8, 10, 12, 24, 32, 64, 100, 128, 256])
def test_attention_block_sizes(block, d, dtype):
    b = Batch([(700, 1), (130, 70), (0, 11), (255, 1), (13, 0)], 8, 2, d, block, dtype, seed=block)
    b.check(b.run())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d,heads,kv_heads", [(32, 4, 2), (80, 4, 1), (96, 3, 3), (256, 2, 1), (2, 2, 2), (33, 2, 1),
                                              (64, 130, 1), (128, 300, 2), (64, 128, 1), (128, 127, 1)])
def test_attention_other_shapes(d, heads, kv_heads, dtype):
    b = Batch([(100, 1), (20, 15), (0, 3)], heads, kv_heads, d, 16, dtype, seed=d)
    b.check(b.run())


@pytest.mark.parametrize("d", [64, 128])
def test_attention_many_sequences(d):
    rs = np.random.RandomState(3)
    b = Batch([(int(rs.randint(0, 90)), int(rs.choice([0, 1, 1, 1, 9]))) for _ in range(1300)], 4, 2, d, 16, F16)
    b.check(b.run())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_attention_long_context(dtype):
    b = Batch([(31000, 1), (30000, 33), (9, 2)], 32, 8, 128, 64, dtype)
    b.check(b.run())


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16), (96, F16)])
def test_attention_rows_without_a_sequence_stay(d, dtype):
    b = Batch([(40, 3), (0, 0), (7, 1)], 4, 2, d, 16, dtype, first_row=2, tail_rows=4)
    out = torch.full_like(b.q, 7.0)
    got = b.run(out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (got[:2] == 7).all() and (got[-4:] == 7).all()
    b.check(got)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16), (96, F16)])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), 6e4])
def test_attention_pages_behind_the_end_hold_anything(d, dtype, junk):
    """Rows of a page behind a sequence's end, and pages no table names."""
    b = Batch([(40, 1), (130, 17), (0, 3), (127, 1), (250, 5)], 4, 2, d, 24, dtype)
    for s in range(5):
        ln = b.pre[s] + b.new[s]
        last = int(b.table[s, (ln - 1) // 24])
        b.pool[last, :, :, :, (ln - 1) % 24 + 1:] = junk
    b.pool[torch.as_tensor(b.unused).cuda()] = junk
    b.check(b.run())


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16), (96, F16)])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf")])
def test_attention_later_rows_do_not_reach_earlier_ones(d, dtype, where, junk):
    """A token whose K or V overflowed: the rows before it are what they are without it."""
    b = Batch([(100, 90), (3, 40), (0, 140)], 8, 2, d, 16, dtype)
    want = b.want()
    pos = [150, 20, 77]
    for s, p in enumerate(pos):
        blk = int(b.table[s, p // 16])
        b.pool[blk, :, 0 if where == "k" else 1, 1, p % 16, 5] = junk
    got = b.run()
    for s, p in enumerate(pos):
        a, i = int(b.qs[s]), p - b.pre[s]
        want[a + i:a + b.new[s], 4:] = float("nan")          # the second kv head's rows that see it
        seen = got[a + i:a + b.new[s], 4:]
        if where == "v":                                     # only that column
            assert not torch.isfinite(seen[..., 5]).any()
            assert torch.isfinite(seen[..., :5]).all() and torch.isfinite(seen[..., 6:]).all()
    b.check(got, want)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_attention_q_scales(d, dtype):
    """Queries of any size: the two fp16 terms are relative to the row's largest."""
    for scale in (1e-30, 1e-6, 1e3, 1e6):
        b = Batch([(70, 9), (300, 1)], 4, 2, d, 16, dtype, q_scale=scale)
        if scale > 1:
            b.pool[:, :, 0] = (b.pool[:, :, 0].float() * (2.0 / scale)).to(dtype)
        want = b.want()
        got = b.run()
        if scale < 1e5:
            b.check(got, want)
        else:                                                # fp16 K becomes subnormal: what is left of it counts
            assert float((got.double() - want).norm() / want.norm()) < 1e-5


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (128, BF16)])
def test_attention_large_v(d, dtype):
    b = Batch([(300, 40), (90, 1)], 4, 2, d, 16, dtype)
    b.pool[:, :, 1] = (b.pool[:, :, 1].float() * 1e4).to(dtype)
    b.check(b.run())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("k_size,v_sizes", [(1.0, [1e-3, 1.0, 0.0, 1e-2]), (1e-3, [1e5, 1.0]), (1.0, [1e-30]), (1e8, [1e30, 1e28]),
                                            (1e-12, [3e4, 1e-4, 1e-6]), (1.0, [0.0]), (0.0, [1.0])])
def test_attention_bf16_magnitudes(d, k_size, v_sizes):
    """bf16 pages far outside of fp16's range, other pages beside them."""
    b = Batch([(700, 40), (130, 1), (5, 9)], 4, 2, d, 16, BF16)
    for i in range(b.pool.shape[0]):
        b.pool[i, :, 0] *= k_size * (1.0, 0.5)[i % 2]
        b.pool[i, :, 1] *= v_sizes[i % len(v_sizes)]
    if k_size:
        b.q *= min(1.0 / k_size, 1e6)
    b.check(b.run())


@pytest.mark.parametrize("d", [64, 128, 96])
def test_attention_missing_pages(d):
    b = Batch([(100, 3), (50, 1), (10, 2)], 4, 2, d, 16, F16)
    want = b.want()
    good, b.table = b.table, b.table.clone()
    b.table[0, 2] = 10 ** 6
    b.table[1] = -1
    f = new_flags()
    got = b.run(flags=f)
    b.table = good                                           # the plain form never sees the bad entries
    assert int(f) == BAD_BLOCK
    assert (got[3] == 0).all()                               # no page left: zeros
    on = torch.ones(103, dtype=torch.bool, device="cuda")
    on[32:48] = False                                        # the missing page's keys
    k, v = b.seq(0).repeat_interleave(b.g, 1)[:, :, on]
    x = torch.einsum("nhd,hkd->hnk", b.q[:3].double(), k) / d ** 0.5
    hide = torch.ones(3, 87, dtype=torch.bool, device="cuda").triu(85)
    want[:3] = torch.einsum("hnk,hkd->nhd", torch.softmax(x.masked_fill(hide, float("-inf")), -1), v)
    want[3] = 0
    b.check(got, want)


@pytest.mark.parametrize("d", [64, 96])
def test_attention_bad_lengths(d):
    b = Batch([(20, 3), (5, 2), (8, 1)], 4, 2, d, 16, F16)
    want = b.want()
    f = new_flags()
    b.prefix[1] = 10 ** 6                                    # past its table
    got = b.run(flags=f)
    assert int(f) == BAD_LENGTH
    want[3:5] = float("nan")
    ok = ~torch.isnan(want)
    assert float((got.double() - want)[ok].abs().max()) < 1e-3
    b.prefix[1] = -4
    f.zero_()
    b.run(flags=f)
    assert int(f) == BAD_LENGTH
    b.prefix[1] = 5
    b.max_q = 2                                              # a bound that is too small: rows past it stay
    f.zero_()
    out = torch.full_like(b.q, 7.0)
    b.run(flags=f, out=out)
    assert int(f) == BAD_LENGTH and (out[2] == 7).all()


def test_attention_unaligned_tensors():
    b = Batch([(100, 5), (33, 1)], 4, 2, 64, 16, F16)
    want = b.want()
    q = torch.empty(b.q.numel() + 1, device="cuda")[1:].view_as(b.q).copy_(b.q)
    pool = torch.empty(b.pool.numel() + 1, dtype=F16, device="cuda")[1:].view_as(b.pool).copy_(b.pool)
    out = torch.empty(b.q.numel() + 3, device="cuda")[3:].view_as(b.q)
    b.check(kv.cache_attention(q, b.pool, 0, b.table, b.q_start, b.prefix, 5, 105), want)
    b.check(kv.cache_attention(b.q, pool, 0, b.table, b.q_start, b.prefix, 5, 105), want)
    b.check(kv.cache_attention(b.q, b.pool, 0, b.table, b.q_start, b.prefix, 5, 105, out=out), want)


@pytest.mark.parametrize("block", [16, 10])
def test_attention_offsets_past_32_bits(block):
    """Pages whose elements lie past 2^32 bytes and past 2^31 elements of the pool."""
    b = Batch([(300, 20), (77, 1)], 8, 8, 128, block, F16)
    nb = (1 << 31) // (2 * 8 * block * 128) + 600
    pool = torch.empty((nb, 1, 2, 8, block, 128), dtype=F16, device="cuda")
    n = b.pool.shape[0]
    pool[nb - n:] = b.pool
    want = b.want()
    got = kv.cache_attention(b.q, pool, 0, b.table + (nb - n), b.q_start, b.prefix, 20, 320)
    b.check(got, want)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_attention_is_the_same_in_every_run(d, dtype):
    b = Batch([(3000, 1), (700, 260), (0, 50)], 8, 2, d, 16, dtype)
    first = b.run().clone()
    for _ in range(5):
        assert torch.equal(b.run(), first)


def test_attention_agrees_with_the_fp32_pool():
    b = Batch([(400, 30), (90, 1)], 14, 2, 64, 16, F16)
    out = torch.empty_like(b.q)
    paged_attention(b.q, b.pool.float(), 0, b.table, b.q_start, b.prefix, b.max_q, b.max_total, out)
    b.check(b.run(), out.double())


@pytest.mark.parametrize("d", [64, 128])
def test_attention_streams_and_graphs(d):
    b = Batch([(600, 1), (90, 1), (300, 1)], 8, 2, d, 16, F16)
    b.check(b.run())
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for s in (s1, s2):
        with torch.cuda.stream(s):
            outs.append(b.run())
    torch.cuda.synchronize()
    for o in outs:
        b.check(o)
    # two graphs of one capture stream, replayed at once with other lengths
    graphs, gouts = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gouts.append(b.run())
        graphs.append(g)
    b.prefix.copy_(i32([555, 12, 299]))
    b.pre = [555, 12, 299]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in gouts:
        b.check(o)


# --------------------------------------------------------------------------- #
# write
# --------------------------------------------------------------------------- #

def tables(d, n=600, theta=10000.0):
    ang = torch.outer(torch.arange(n).double(), theta ** (-torch.arange(0, d, 2).double() / d))
    return ang.cos().float().cuda(), ang.sin().float().cuda()


def write_case(T, hq, hkv, d, block, dtype, norm, seed=0, layers=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed)
    nb = T // block + 3
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g, device="cuda") * 1.5
    pool = torch.randn(nb, layers, 2, hkv, block, d, generator=g, device="cuda").to(dtype)
    slots = rs.permutation(nb * block)[:T]
    pos = rs.randint(0, 600, T)
    nq = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if norm & 1 else None
    nk = 1 + 0.1 * torch.randn(d, generator=g, device="cuda") if norm & 2 else None
    return qkv, pool, i64(pos), i64(slots), nq, nk


def split_heads(qkv, hq, hkv, d):
    return qkv.view(-1, hq + 2 * hkv, d).split([hq, hkv, hkv], 1)


def turn(x, c, s):
    d = x.shape[-1] // 2
    a, b = x[..., :d], x[..., d:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("T,hq,hkv,d,block", [(1, 14, 2, 64, 16), (37, 32, 8, 128, 16), (5, 4, 2, 64, 1), (300, 3, 1, 128, 24),
                                              (9, 4, 2, 96, 7), (3, 2, 2, 2, 4), (2, 2, 1, 256, 16)])
def test_write_without_norms_is_torchs_bits(T, hq, hkv, d, block, dtype):
    qkv, pool, pos, slots, _, _ = write_case(T, hq, hkv, d, block, dtype, 0)
    cos, sin = tables(d)
    want = pool.clone()
    q, k, v = split_heads(qkv, hq, hkv, d)
    c, s = cos[pos][:, None], sin[pos][:, None]
    want[slots // block, 1, 0, :, slots % block] = turn(k, c, s).to(dtype)
    want[slots // block, 1, 1, :, slots % block] = v.to(dtype)
    f = new_flags()
    got = kv.rope_cache_write(qkv, pool, 1, pos, slots, cos, sin, flags=f)
    assert int(f) == 0
    assert torch.equal(got, turn(q, c, s)) and torch.equal(pool, want)
    if dtype is F32:
        ref, q2 = pool.clone().normal_(), torch.empty_like(got)
        ref2 = ref.clone()
        kv.rope_cache_write(qkv, ref, 0, pos, slots, cos, sin)
        _lib.call("ksh_rope_kv_write", qkv.data_ptr(), T, hq, hkv, d, pos.data_ptr(), slots.data_ptr(), cos.data_ptr(),
                  sin.data_ptr(), cos.shape[0], q2.data_ptr(), ref2.data_ptr(), pool.shape[0], 2, 0, block, f.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(ref, ref2) and torch.equal(got, q2)


@pytest.mark.parametrize("norm", [1, 2, 3])
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("T,hq,hkv,d,block", [(1, 14, 2, 64, 16), (65, 32, 8, 128, 16), (7, 5, 1, 96, 10), (300, 3, 3, 64, 64)])
def test_write_with_norms(T, hq, hkv, d, block, dtype, norm):
    qkv, pool, pos, slots, nq, nk = write_case(T, hq, hkv, d, block, dtype, norm)
    qkv[0] *= 1e-4                                           # eps counts there
    cos, sin = tables(d)
    before = pool.clone()
    q, k, v = (x.double() for x in split_heads(qkv, hq, hkv, d))
    c, s = cos[pos][:, None].double(), sin[pos][:, None].double()

    def normed(x, w):
        return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()

    def size(x):
        y = x.abs()
        return torch.cat([y[..., :d // 2] + y[..., d // 2:]] * 2, -1)

    got = kv.rope_cache_write(qkv, pool, 0, pos, slots, cos, sin, q_norm=nq, k_norm=nk, eps=1e-6)
    yq, yk = normed(q, nq), normed(k, nk)
    bound = 16 * 2.0 ** -24
    assert ((got.double() - turn(yq, c, s)).abs() <= bound * size(yq)).all()
    gk = pool[slots // block, 0, 0, :, slots % block].double()
    want = turn(yk, c, s)
    half = torch.finfo(dtype).eps / 2 * (want.abs() + bound * size(yk)) + torch.finfo(dtype).smallest_normal
    assert ((gk - want).abs() <= bound * size(yk) + half).all()
    assert torch.equal(pool[slots // block, 0, 1, :, slots % block], v.float().to(dtype))
    pool[slots // block, 0, :, :, slots % block] = before[slots // block, 0, :, :, slots % block]
    assert torch.equal(pool, before)                         # nothing else was touched


@pytest.mark.parametrize("d", [64, 96])
def test_write_bad_slots_and_positions(d):
    qkv, pool, pos, slots, _, _ = write_case(6, 4, 2, d, 8, F16, 0)
    cos, sin = tables(d)
    before = pool.clone()
    slots[2], slots[3] = -1, pool.shape[0] * 8
    f = new_flags()
    kv.rope_cache_write(qkv, pool, 0, pos, slots, cos, sin, flags=f)
    assert int(f) == BAD_SLOT
    on = torch.ones(pool.shape[0] * 8, dtype=torch.bool, device="cuda")
    on[slots[[0, 1, 4, 5]]] = False
    same = (pool == before).all(-1).all(3).all(2).all(1).reshape(-1)       # [nb * block]
    assert same[on].all()
    pos[1] = 600
    pos[4] = -1
    f.zero_()
    slots[2], slots[3] = slots[0] // 8 * 8 + (slots[0] + 1) % 8, -1
    got = kv.rope_cache_write(qkv, pool, 0, pos, slots, cos, sin, flags=f)
    assert int(f) == BAD_SLOT | BAD_POSITION
    q, _, _ = split_heads(qkv, 4, 2, d)
    assert torch.equal(got[1], q[1]) and torch.equal(got[4], q[4])         # position 0 turns nothing


def test_write_overflow_and_unaligned():
    qkv, pool, pos, slots, _, _ = write_case(4, 4, 2, 64, 8, F16, 0)
    cos, sin = tables(64)
    qkv[1, -3] = 1e6                                          # past fp16: infinite, as torch rounds
    qkv[2, -3] = float("nan")
    kv.rope_cache_write(qkv, pool, 0, pos, slots, cos, sin)
    got = pool[slots // 8, 0, 1, :, slots % 8]
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(split_heads(qkv, 4, 2, 64)[2].to(F16)))
    p2, x2 = torch.zeros_like(pool), torch.empty(qkv.numel() + 1, device="cuda")[1:].view_as(qkv).copy_(qkv)
    kv.rope_cache_write(x2, p2, 0, pos, slots, cos, sin)
    assert torch.equal(torch.nan_to_num(p2[slots // 8, 0, :, :, slots % 8]),
                       torch.nan_to_num(pool[slots // 8, 0, :, :, slots % 8]))


# --------------------------------------------------------------------------- #
# pages
# --------------------------------------------------------------------------- #

def fork_want(pool, table, lens, parents, refs):
    """The definition, one child after the other, on the host."""
    pool, table, refs = pool.clone(), table.tolist(), refs.tolist()
    b, m = pool.shape[4], len(table[0])
    for row, ln in zip(table, lens):
        for page in row[:-(-ln // b)]:
            refs[page] -= 1
    out, want, seen = [], [], set()
    for i, p in enumerate(parents):
        row = [0] * m
        if p >= 0:
            full, rest = lens[p] // b, lens[p] % b
            row[:full] = table[p][:full]
            for page in row[:full]:
                refs[page] += 1
            if full < m:
                if rest and p not in seen:
                    row[full] = table[p][full]
                    refs[row[full]] += 1
                    seen.add(p)
                else:
                    want.append(i)
        out.append(row)
    free = [i for i, r in enumerate(refs) if r == 0]
    ok = set()
    for i, page in zip(want, free):
        p = parents[i]
        full, rest = lens[p] // b, lens[p] % b
        out[i][full] = page
        refs[page] = 1
        ok.add(i)
        pool[page, :, :, :, :rest] = pool[table[p][full], :, :, :, :rest]
    slots = [-1 if p < 0 or lens[p] // b >= m or (i in want and i not in ok) else out[i][lens[p] // b] * b + lens[p] % b
             for i, p in enumerate(parents)]
    return out, [0 if p < 0 else lens[p] for p in parents], slots, refs, pool


def fork_case(lens, m, block, nb, kv_heads=2, d=64, layers=3, dtype=F16, shared=True, seed=0):
    """Sequences whose first pages are shared in pairs."""
    rs = np.random.RandomState(seed)
    ids = list(rs.permutation(nb))
    table, refs = np.zeros((len(lens), m), np.int64), np.zeros(nb, np.int64)
    for s, ln in enumerate(lens):
        held = -(-ln // block)
        for j in range(held):
            if shared and s % 2 and j < ln // block and j < lens[s - 1] // block:
                table[s, j] = table[s - 1, j]
            else:
                table[s, j] = ids.pop()
            refs[table[s, j]] += 1
    refs[ids.pop()] = 2                                      # held by someone else
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = torch.randn(nb, layers, 2, kv_heads, block, d, generator=g, device="cuda").to(dtype)
    return pool, i32(table), lens, i32(refs)


def check_fork(case, parents, want_flags=0):
    pool, table, lens, refs = case
    want = fork_want(pool, table, lens, parents, refs)
    f = new_flags()
    old = (table.clone(), refs.clone())
    got = kv.fork_pages(pool, table, i32(lens), i32(parents).view(-1), refs, flags=f)
    assert int(f) == want_flags
    assert torch.equal(table, old[0]) and torch.equal(refs, old[1])
    for x, y in zip(got, want):
        assert x.tolist() == y
    assert torch.equal(pool, want[4])
    return got


@pytest.mark.parametrize("lens,parents", [
    ([37], [0]), ([37], [0, 0, 0, 0]), ([32], [0, 0]), ([0], [0, 0]), ([1, 16, 15], [2, 1, 0, 0, 1, 2, 2]),
    ([37, 40, 64, 33, 90, 10], [0, 0, 2, 2, 2, -1, 4, 4]), ([37, 40], [-1, -1]), ([37, 40], []),
    ([50] * 16, [3] * 40), (list(range(0, 120, 3)), list(range(40))), (list(range(0, 120, 3)), [7, 39, 0, 7, 21, 39, -1, 7]),
], ids=lambda x: None)
@pytest.mark.parametrize("block", [16, 10])
def test_fork(lens, parents, block):
    check_fork(fork_case(lens, 14, block, 600), parents)


@pytest.mark.parametrize("dtype,d,kv_heads,block", [(BF16, 128, 8, 16), (F32, 64, 2, 24), (F16, 3, 1, 5), (F16, 2, 3, 7),
                                                    (F16, 4, 1, 3), (F32, 1, 1, 2), (BF16, 256, 1, 1)])
def test_fork_types_and_sizes(dtype, d, kv_heads, block):
    check_fork(fork_case([11, 23, 9, 30], 40, block, 200, kv_heads, d, 2, dtype), [0, 0, 1, 1, 1, 3, 2, 2, 0])


def test_fork_many():
    rs = np.random.RandomState(1)
    lens = [int(x) for x in rs.randint(0, 200, 1500)]
    parents = [int(x) for x in rs.randint(-1, 1500, 5000)]
    check_fork(fork_case(lens, 26, 8, 40000, 1, 8, 1), parents)


def test_fork_reuses_freed_pages_and_runs_out():
    # 4 pages used of 5 (one held elsewhere): a fork that frees two sequences takes their pages
    case = fork_case([16, 32, 16], 4, 16, 5, shared=False)
    check_fork(case, [1, 1])
    case = fork_case([20, 20], 4, 16, 6, shared=False)
    check_fork(case, [0, 0, 0, 0, 1], NO_PAGE)


def test_fork_bad_input():
    pool, table, lens, refs = fork_case([20, 20, 64], 4, 16, 40)
    f = new_flags()
    t, ln, slots, r = kv.fork_pages(pool, table, i32(lens), i32([2, 0]), refs, flags=f)
    assert int(f) == BAD_LENGTH and slots.tolist()[0] == -1 and slots.tolist()[1] >= 0       # 64 tokens fill the row
    f.zero_()
    t, ln, slots, r = kv.fork_pages(pool, table, i32(lens), i32([3, 0, 10 ** 6]), refs, flags=f)
    assert int(f) == BAD_PARENT and slots.tolist()[0] == -1 and slots.tolist()[2] == -1 and t[0].tolist() == [0] * 4
    f.zero_()
    kv.fork_pages(pool, table, i32([20, 65, -1]), i32([0]), refs, flags=f)
    assert int(f) & BAD_LENGTH
    f.zero_()
    table[1, 1] = 40
    before = pool.clone()
    t, ln, slots, r = kv.fork_pages(pool, table, i32([20, 20, 64]), i32([1, 1]), refs, flags=f)
    assert int(f) & BAD_BLOCK and slots[0] == -1
    free = [int(t[1, 1])]
    before[free] = pool[free]
    assert torch.equal(pool, before)
    f.zero_()
    kv.fork_pages(pool, table[:1].contiguous(), i32([20]), i32([0]), torch.zeros_like(refs), flags=f)
    assert int(f) & BAD_BLOCK                                # held more often than counted


def compact_want(pool, table, refs):
    pool, refs, nb = pool.clone(), refs.tolist(), pool.shape[0]
    used = [i for i in range(nb) if refs[i] > 0]
    u = len(used)
    to = list(range(nb))
    for src, dst in zip([i for i in used if i >= u], [i for i in range(u) if refs[i] <= 0]):
        to[src] = dst
    new = [0] * nb
    for i in used:
        new[to[i]] = refs[i]
        if to[i] != i:
            pool[to[i]] = pool[i]
    return [[to[x] if 0 <= x < nb else x for x in row] for row in table.tolist()], new, to, [u], pool


@pytest.mark.parametrize("nb,used,dtype,d,block", [
    (1, 0, F16, 64, 16), (1, 1, F16, 64, 16), (2, 1, F16, 64, 16), (60, 31, F16, 64, 16), (60, 60, F16, 64, 16),
    (60, 0, BF16, 64, 16), (333, 100, BF16, 128, 24), (500, 499, F32, 64, 10), (129, 64, F16, 3, 5), (33, 7, F16, 2, 1),
    (9000, 5000, F16, 8, 2), (40000, 300, F16, 4, 1), (4097, 4000, F16, 6, 1)])
def test_compact(nb, used, dtype, d, block):
    rs = np.random.RandomState(nb)
    g = torch.Generator(device="cuda").manual_seed(nb)
    ids = rs.permutation(nb)[:used]
    refs = np.zeros(nb, np.int64)
    refs[ids] = rs.randint(1, 5, used)
    table = rs.randint(-1, nb + 1, (7, 13))
    pool = torch.randn(nb, 2, 2, 2, block, d, generator=g, device="cuda").to(dtype)
    table, refs = i32(table), i32(refs)
    want = compact_want(pool, table, refs)
    got = kv.compact_pages(pool, table, refs)
    for x, y in zip(got, want):
        assert x.tolist() == y
    # what moved away stays where it was; everything in use is at its new place
    assert torch.equal(pool, want[4])


@pytest.mark.parametrize("lowest", [True, False])
def test_compact_where_the_used_pages_lie(lowest):
    refs = [0] * 100
    for i in range(40):
        refs[i if lowest else 99 - i] = 1
    pool = torch.randn(100, 1, 2, 1, 4, 8, device="cuda").half()
    table = i32([[5, 99, 70]])
    want = compact_want(pool, table, i32(refs))
    got = kv.compact_pages(pool, table, i32(refs))
    for x, y in zip(got, want):
        assert x.tolist() == y
    assert torch.equal(pool, want[4])


def test_pages_in_a_graph():
    pool, table, lens, refs = fork_case([37, 40, 64, 33], 8, 16, 100)
    ln, parents = i32(lens), i32([0, 0, 2, 3, 3])
    want = fork_want(pool, table, lens, [0, 0, 2, 3, 3], refs)
    base = pool.clone()
    kv.fork_pages(pool, table, ln, parents, refs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t, n, slots, r = kv.fork_pages(pool, table, ln, parents, refs)
        t2, r2, m, u = kv.compact_pages(pool, t, r)
    for _ in range(2):
        pool.copy_(base)
        g.replay()
    torch.cuda.synchronize()
    assert t.tolist() == want[0] and r.tolist() == want[3] and slots.tolist() == want[2]
    want2 = compact_want(want[4], t, r)
    assert t2.tolist() == want2[0] and r2.tolist() == want2[1] and m.tolist() == want2[2]
    assert torch.equal(pool, want2[4])


# --------------------------------------------------------------------------- #
# refusals
# --------------------------------------------------------------------------- #

def test_refusals():
    b = Batch([(20, 3)], 4, 2, 64, 16, F16)
    args = [b.q, b.pool, 0, b.table, b.q_start, b.prefix, 3, 23]

    def refused(i, x, kind=ValueError):
        a = list(args)
        a[i] = x
        with pytest.raises(kind):
            kv.cache_attention(*a)
    refused(0, b.q.half())
    refused(0, b.q.transpose(0, 1))
    refused(0, b.q[:, :3].contiguous())                      # heads not a multiple
    refused(0, b.q.cpu(), _lib.KshipraLibraryError)
    refused(1, b.pool.float())
    refused(1, b.pool[:, :, :1].contiguous())
    refused(1, b.pool.transpose(3, 4))
    refused(1, b.pool.cpu(), _lib.KshipraLibraryError)
    refused(2, 1)
    refused(2, -1)
    refused(3, b.table.long())
    refused(4, b.q_start[:1])
    refused(5, b.prefix.long())
    refused(6, -1)
    refused(7, -1)
    with pytest.raises(ValueError):
        kv.cache_attention(*args, out=torch.empty(3, 4, 32, device="cuda"))
    big = torch.zeros(1, 1, 2, 1, 16, 512, dtype=F16, device="cuda")
    with pytest.raises(_lib.KshipraLibraryError):
        kv.cache_attention(torch.zeros(3, 4, 512, device="cuda"), big, 0, b.table, b.q_start, b.prefix, 3, 23)
    qkv, pool, pos, slots, nq, _ = write_case(3, 4, 2, 64, 8, F16, 1)
    cos, sin = tables(64)
    for bad in ([qkv[:, :-1], pool, 0, pos, slots, cos, sin], [qkv, pool, 2, pos, slots, cos, sin],
                [qkv, pool.double(), 0, pos, slots, cos, sin], [qkv, pool, 0, pos[:2], slots, cos, sin],
                [qkv, pool, 0, pos.int(), slots, cos, sin], [qkv, pool, 0, pos, slots, cos[:, :5], sin],
                [qkv[:, :256].contiguous(), pool, 0, pos, slots, cos, sin]):
        with pytest.raises(ValueError):
            kv.rope_cache_write(*bad)
    with pytest.raises(ValueError):
        kv.rope_cache_write(qkv, pool, 0, pos, slots, cos, sin, q_norm=nq[:10])
    pool, table, lens, refs = fork_case([20, 20], 4, 16, 40)
    for bad in ([pool, table.long(), i32(lens), i32([0]), refs], [pool, table, i32([20]), i32([0]), refs],
                [pool, table, i32(lens), i32([[0]]), refs], [pool, table, i32(lens), i32([0]), refs[:5]],
                [pool.transpose(0, 1), table, i32(lens), i32([0]), refs]):
        with pytest.raises(ValueError):
            kv.fork_pages(*bad)
    with pytest.raises(ValueError):
        kv.compact_pages(pool, table, refs[:5])
    with pytest.raises(_lib.KshipraLibraryError):
        kv.compact_pages(pool.cpu(), table, refs)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16), (96, F16)])
def test_attention_without_any_new_token(d, dtype):
    b = Batch([(50, 0), (0, 0), (7, 0)], 4, 2, d, 16, dtype, tail_rows=3)
    f = new_flags()
    out = torch.full_like(b.q, 7.0)
    kv.cache_attention(b.q, b.pool, 0, b.table, b.q_start, b.prefix, 5, 60, out=out, flags=f)
    assert (out == 7).all() and int(f) == 0


@pytest.mark.parametrize("d", [64, 128])
def test_attention_bf16_values_near_the_largest(d):
    """Sums stay in range where the values nearly fill it."""
    b = Batch([(40, 3), (9, 1)], 4, 2, d, 16, BF16)
    b.pool[:, :, 1] = (b.pool[:, :, 1].float().abs().clamp(max=3.0) * 2.0 ** 118).to(BF16)
    b.q *= 8.0                                               # the maximum rises as tiles go by
    want = b.want()
    got = b.run().double()
    assert float((got - want).abs().max() / want.abs().max()) < 1e-5


def test_attention_loose_bounds():
    """max_q_len and max_total_len far above what comes."""
    for d in (64, 96):
        b = Batch([(40, 3), (9, 1)], 4, 2, d, 16, F16)
        b.max_q, b.max_total = 2 ** 31 - 1, 2 ** 40
        b.check(b.run())


def test_fork_from_nothing():
    pool = torch.randn(6, 1, 2, 1, 4, 8, device="cuda").half()
    none = torch.empty((0, 3), dtype=torch.int32, device="cuda")
    refs = i32([1, 0, 0, 2, 0, 0])
    f = new_flags()
    t, n, s, r = kv.fork_pages(pool, none, i32([]), i32([-1, -1]), refs, flags=f)
    assert t.tolist() == [[0] * 3] * 2 and n.tolist() == [0, 0] and s.tolist() == [-1, -1] and torch.equal(r, refs)
    assert int(f) == 0


def test_two_calls_at_once_on_two_streams():
    """Forks and attentions of two batches on streams of their own."""
    bs = [Batch([(300, 20), (77, 1)], 8, 2, 128, 16, F16, seed=i) for i in range(2)]
    cases = [fork_case([37, 40, 64, 33], 8, 16, 100, seed=i) for i in range(2)]
    wants = [fork_want(c[0], c[1], c[2], [0, 0, 2, 3, 3], c[3]) for c in cases]
    lens, parents = i32([37, 40, 64, 33]), i32([0, 0, 2, 3, 3])
    torch.cuda.synchronize()
    streams, got, forked = [torch.cuda.Stream() for _ in range(2)], [], []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, bs[i].run()))
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            forked.append(kv.fork_pages(cases[i][0], cases[i][1], lens, parents, cases[i][3]))
    torch.cuda.synchronize()
    for i, out in got:
        bs[i].check(out)
    for c, f, w in zip(cases, forked, wants):
        for x, y in zip(f, w):
            assert x.tolist() == y
        assert torch.equal(c[0], w[4])


def test_empty_calls():
    b = Batch([(20, 3)], 4, 2, 64, 16, F16)
    none = b.q[:0].contiguous()
    assert kv.cache_attention(none, b.pool, 0, b.table, i32([0, 0]), b.prefix, 3, 23).shape[0] == 0
    out = torch.full_like(b.q, 7.0)
    kv.cache_attention(b.q, b.pool, 0, b.table[:0].contiguous(), i32([0]), i32([]), 3, 23, out=out)
    assert (out == 7).all()
    cos, sin = tables(64)
    assert kv.rope_cache_write(torch.empty(0, 512, device="cuda"), b.pool, 0, i64([]), i64([]), cos, sin).shape[0] == 0
    t, n, s, r = kv.fork_pages(b.pool, b.table, i32([23]), i32([]), i32([1] * b.pool.shape[0]))
    assert t.shape[0] == 0 and r.sum() == b.pool.shape[0] - 2


def shared_fork_want(pool, table, lens, parents, refs):
    """fork_want where rows may hold the same page while it fills: it stays with the
    first child that continues in it if nobody else is left to hold it."""
    pool, table, refs = pool.clone(), table.tolist(), refs.tolist()
    b, m = pool.shape[4], len(table[0])
    for row, ln in zip(table, lens):
        for page in row[:-(-ln // b)]:
            refs[page] -= 1
    out = [[0] * m if p < 0 else table[p][:lens[p] // b] + [0] * (m - lens[p] // b) for p in parents]
    for i, p in enumerate(parents):
        for page in [] if p < 0 else table[p][:lens[p] // b]:
            refs[page] += 1
    last = [-1 if p < 0 or lens[p] // b >= m else lens[p] // b for p in parents]
    kept = {}
    for i, p in enumerate(parents):
        if last[i] >= 0 and lens[p] % b and refs[table[p][last[i]]] == 0:
            kept.setdefault(table[p][last[i]], i)
    for page, i in kept.items():
        refs[page], out[i][last[i]] = 1, page
    free = iter([i for i, r in enumerate(refs) if r == 0])
    for i, p in enumerate(parents):
        if last[i] >= 0 and i not in kept.values():
            page, rest = next(free), lens[p] % b
            refs[page], out[i][last[i]] = 1, page
            pool[page, :, :, :, :rest] = pool[table[p][last[i]], :, :, :, :rest]
    slots = [-1 if last[i] < 0 else out[i][last[i]] * b + lens[p] % b for i, p in enumerate(parents)]
    return out, [0 if p < 0 else lens[p] for p in parents], slots, refs, pool


@pytest.mark.parametrize("lens,parents,outside", [
    ([37, 37, 37, 37], [0, 1, 2, 3], 0), ([37, 37, 37, 37], [3, 1, 1, 0, 2], 0), ([37], [0], 1), ([37], [0, 0], 1),
    ([37, 37], [1], 0), ([37, 48, 37], [1, 0, 2], 0), ([37, 48, 41], [0, 2], 0), ([37, 48], [-1, 0], 2), ([37, 35], [1, 0, 0], 0),
], ids=lambda x: None)
def test_fork_of_pages_that_several_rows_fill(lens, parents, outside):
    """Rows of one prompt, repeated: no two children write into one page."""
    row = [5, 9, 2, 0]
    table = i32([row] * len(lens))
    refs = [0] * 24
    for ln in lens:
        for page in row[:-(-ln // 16)]:
            refs[page] += 1
    refs[2] += outside
    refs = i32(refs)
    pool = torch.randn(24, 2, 2, 2, 16, 64, generator=torch.Generator("cuda").manual_seed(0), device="cuda").half()
    want = shared_fork_want(pool, table, lens, parents, refs)
    f = new_flags()
    got = kv.fork_pages(pool, table, i32(lens), i32(parents), refs, flags=f)
    assert int(f) == 0
    for x, y in zip(got, want):
        assert x.tolist() == y
    assert torch.equal(pool, want[4])
    slots = [s for s in got[2].tolist() if s >= 0]
    assert len({s // 16 for s in slots}) == len(slots)


def test_two_threads_on_one_stream():
    """Each call's launches stay together: both use the stream's workspace."""
    bs = [Batch([(5000 + 900 * i, 20), (77, 1)], 8, 2, 128, 16, F16, seed=i) for i in range(2)]
    want = [b.run() for b in bs]
    got, stream = [[], []], torch.cuda.current_stream()
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(stream):
            for _ in range(60):
                got[i].append(bs[i].run())

    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 60 and all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d,block", [(255, 7), (256, 16), (130, 16), (12, 1), (1, 3), (80, 24), (112, 10), (134, 64)])
def test_attention_other_dimensions(d, block, dtype):
    """Lengths around the warps' runs of 16 keys and the CTA's of 128, and long ones."""
    b = Batch([(0, 1), (15, 1), (0, 18), (16, 1), (126, 4), (0, 0), (1500, 1), (700, 33), (31, 1)], 6, 2, d, block, dtype, layers=2,
              seed=d, first_row=1, tail_rows=2)
    out = torch.full_like(b.q, 7.0)
    b.run(out=out)
    assert (out[:1] == 7).all() and (out[-2:] == 7).all()
    b.check(out)
    assert torch.equal(b.run()[1:-2], out[1:-2])


def test_attention_other_dimensions_many_sequences():
    rs = np.random.RandomState(4)
    b = Batch([(int(rs.randint(0, 90)), int(rs.choice([0, 1, 1, 1, 9]))) for _ in range(700)], 4, 2, 96, 16, F16)
    b.check(b.run())
    f = new_flags()
    b.prefix[[3, 699]] = -1
    b.run(flags=f)
    assert int(f) == BAD_LENGTH


# ---- few rows a sequence: a path of their own (rows = tokens x heads of a group up to 16) ----

FEW = [[(0, 1)], [(540, 1)], [(15, 1), (16, 1), (31, 1), (0, 1), (63, 1), (64, 1), (65, 1)], [(4100, 1), (0, 1), (0, 0), (900, 1)],
       [(3, 2), (0, 2), (500, 1), (2000, 2), (0, 0), (14, 2), (15, 2), (0, 0)], [(int(x), 1) for x in range(0, 1200, 9)],
       [(20000, 1)], [(0, 0), (0, 0), (77, 1)]]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d,heads,kv_heads,block", [(64, 14, 2, 16), (128, 32, 8, 16), (128, 8, 8, 10), (64, 8, 1, 64), (128, 3, 1, 1),
                                                    (64, 5, 5, 7)])
@pytest.mark.parametrize("lengths", range(len(FEW)))
def test_few_rows(lengths, d, heads, kv_heads, block, dtype):
    b = Batch(FEW[lengths], heads, kv_heads, d, block, dtype, layers=2, seed=lengths, first_row=1, tail_rows=2)
    out = torch.full_like(b.q, 7.0)
    f = new_flags()
    b.run(out=out, flags=f)
    assert int(f) == 0 and (out[:1] == 7).all() and (out[-2:] == 7).all()
    b.check(out)
    assert torch.equal(b.run()[1:-2], out[1:-2])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d,heads,kv_heads,new", [(64, 16, 1, 1), (128, 32, 2, 1), (128, 4, 4, 16), (64, 4, 2, 8), (128, 12, 4, 5),
                                                  (64, 9, 3, 5), (64, 17, 1, 1), (128, 6, 3, 9)])
def test_few_rows_of_several_tokens(d, heads, kv_heads, new, dtype):
    """Groups and chunks that fill the 16 rows, or pass them by one."""
    rs = np.random.RandomState(new)
    b = Batch([(int(rs.randint(0, 700)), int(rs.randint(1, new + 1))) for _ in range(30)] + [(3000, new), (0, new), (16, new)],
              heads, kv_heads, d, 16, dtype, seed=new)
    b.check(b.run())


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf"), 6e4])
def test_few_rows_pages_behind_the_end_hold_anything(d, dtype, junk):
    b = Batch([(40, 1), (130, 2), (0, 3), (127, 1), (250, 4)], 4, 2, d, 24, dtype)
    want = b.want()
    for s, (p, n) in enumerate(zip(b.pre, b.new)):
        end = p + n
        page = int(b.table[s, (end - 1) // 24])
        b.pool[page, :, :, :, (end - 1) % 24 + 1:] = junk
    b.pool[b.unused] = junk
    b.check(b.run(), want)


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (64, BF16), (128, BF16)])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), float("-inf")])
def test_few_rows_later_tokens_do_not_reach_earlier_ones(d, dtype, where, junk):
    """What the last token of each chunk brings is seen by its own row alone."""
    b = Batch([(100, 5), (3, 8), (0, 2), (14, 3)], 4, 2, d, 16, dtype)
    want = b.want()
    last = torch.zeros(b.total, dtype=torch.bool, device="cuda")
    for s, (p, n) in enumerate(zip(b.pre, b.new)):
        end = p + n - 1
        b.pool[int(b.table[s, end // 16]), 0, 0 if where == "k" else 1, :, end % 16, 3] = junk
        last[int(b.qs[s]) + n - 1] = True
    got = b.run()
    want[last] = float("nan")
    diff = (got.double() - want)[~last]
    assert torch.isfinite(got[~last]).all()
    assert float(diff.norm()) <= 1e-5 * float(want[~last].norm())
    if where == "v":
        assert not torch.isfinite(got[last][..., 3]).any() and torch.isfinite(got[last][..., :3]).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_few_rows_missing_pages_and_bad_lengths(d, dtype):
    b = Batch([(100, 3), (50, 1), (10, 2)], 4, 2, d, 16, dtype)
    want = b.want()
    good, b.table = b.table, b.table.clone()
    b.table[0, 2] = 10 ** 6
    b.table[1] = -1
    f = new_flags()
    got = b.run(flags=f)
    b.table = good
    assert int(f) == BAD_BLOCK and (got[3] == 0).all()
    on = torch.ones(103, dtype=torch.bool, device="cuda")
    on[32:48] = False
    k, v = b.seq(0).repeat_interleave(b.g, 1)[:, :, on]
    x = torch.einsum("nhd,hkd->hnk", b.q[:3].double(), k) / d ** 0.5
    hide = torch.ones(3, 87, dtype=torch.bool, device="cuda").triu(85)
    want[:3] = torch.einsum("hnk,hkd->nhd", torch.softmax(x.masked_fill(hide, float("-inf")), -1), v)
    want[3] = 0
    b.check(got, want)
    for bad in (10 ** 6, -4):
        b.prefix[1] = bad
        f.zero_()
        b.run(flags=f)
        assert int(f) == BAD_LENGTH
    b.prefix[1] = 50
    b.max_q = 2                                              # rows past the bound stay
    f.zero_()
    out = torch.full_like(b.q, 7.0)
    b.run(flags=f, out=out)
    assert int(f) == BAD_LENGTH and (out[2] == 7).all()


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, F16), (128, BF16)])
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-6, 1e3])
def test_few_rows_q_scales(d, dtype, scale):
    b = Batch([(70, 1), (1300, 1)], 4, 2, d, 16, dtype, q_scale=scale)
    if scale > 1:
        b.pool[:, :, 0] = (b.pool[:, :, 0].float() * (2.0 / scale)).to(dtype)
    b.check(b.run())


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_few_rows_many_sequences(d, dtype):
    rs = np.random.RandomState(3)
    b = Batch([(int(rs.randint(0, 90)), int(rs.choice([0, 1, 1, 1, 4]))) for _ in range(1300)], 8, 2, d, 16, dtype)
    b.check(b.run())


def test_few_rows_loose_bounds_and_captured():
    b = Batch([(4000, 1), (90, 1), (300, 1)], 8, 2, 128, 16, F16)
    b.check(b.run())
    for b.max_total in (0, 1, 2 ** 40):
        b.check(b.run())
    b.max_total = 4001
    out = torch.empty_like(b.q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.run(out=out)
    for p in ([17, 90, 299], [4000, 0, 5]):
        b.pre = p
        b.prefix.copy_(i32(p))
        out.zero_()
        g.replay()
        b.check(out)


def test_few_rows_offsets_past_32_bits():
    b = Batch([(300, 1), (77, 2)], 8, 8, 128, 16, F16)
    nb = (1 << 31) // (2 * 8 * 16 * 128) + 600
    pool = torch.empty((nb, 1, 2, 8, 16, 128), dtype=F16, device="cuda")
    n = b.pool.shape[0]
    pool[nb - n:] = b.pool
    b.check(kv.cache_attention(b.q, pool, 0, b.table + (nb - n), b.q_start, b.prefix, 2, 301), b.want())


# (the tile kernel with whole and with folded row tiles, the few-row kernel, the general kernel)
LARGEST = [(64, 8, 2, [(600, 40), (3000, 1), (0, 1)]), (128, 4, 4, [(5, 130), (2000, 20)]), (64, 4, 2, [(3000, 1), (40, 1)]),
           (128, 32, 8, [(700, 3), (9000, 1)]), (96, 4, 2, [(1500, 2), (0, 7)]), (33, 2, 1, [(900, 1)])]


@pytest.mark.parametrize("scores", ["equal", "rising", "any"])
@pytest.mark.parametrize("d,heads,kv_heads,seqs", LARGEST)
def test_attention_bf16_means_of_the_largest_values(d, heads, kv_heads, seqs, scores):
    """A mean of values is no larger than they are, however many keys add up to it:
    thousands of keys whose V is bf16's largest, with scores that are all the same,
    that rise by less than what the running reference follows (7.9 powers of two behind
    the first 128 keys), or random ones with signs of V that differ."""
    b = Batch(seqs, heads, kv_heads, d, 16, BF16)
    top = torch.finfo(BF16).max
    if scores == "any":
        b.pool[:, :, 1] = torch.where(b.pool[:, :, 1] > -1.0, top, -top)
    else:
        b.pool[:, :, 1] = top
        b.pool[:, :, 0] = 0.0
        b.q.zero_()
    if scores == "rising":
        b.pool[:, :, 0, :, :, 0] = 1.0
        b.pool[b.table[:, :8].long().reshape(-1), :, 0, :, :, 0] = 0.0      # (a page is one sequence's; spare entries name page 0)
        b.q[:, :, 0] = 7.9 * np.log(2.0) * d ** 0.5
    b.check(b.run())


@pytest.mark.parametrize("d,group", [(80, 1), (64, 129)])
def test_attention_more_sequences_than_one_general_call(d, group):
    """The general kernel's calls are split into runs of sequences: 70000 of them, over a
    few pages that they share, some empty, some of three rows, rows of no sequence before them."""
    S, bs = 70000, 16
    rs = np.random.RandomState(0)
    new = rs.choice([0, 1, 1, 1, 3], S)
    pre = rs.randint(0, 20, S)
    qs = 5 + np.concatenate([[0], np.cumsum(new)])
    table = rs.randint(0, 6, (S, 2))
    g = torch.Generator(device="cuda").manual_seed(0)
    pool = torch.randn(6, 1, 2, 1, bs, d, generator=g, device="cuda").half()
    q = torch.randn(int(qs[-1]) + 2, group, d, generator=g, device="cuda")
    out = torch.full_like(q, 7.0)
    f = new_flags()
    kv.cache_attention(q, pool, 0, i32(table), i32(qs), i32(pre), 3, 32, out=out, flags=f)
    assert int(f) == 0 and (out[:5] == 7).all() and (out[int(qs[-1]):] == 7).all()
    seq = np.repeat(np.arange(S), new)
    last = i64(pre[seq] + np.arange(len(seq)) - (qs[:-1][seq] - 5))
    rows = pool[i64(table)[i64(seq)], 0, :, 0].double()                        # [rows, 2 pages, K / V, bs, d]
    top = float(pool[:, :, 1].abs().max())
    for a in range(0, len(seq), 4096):
        k, v = (rows[a:a + 4096, :, i].reshape(-1, 2 * bs, d) for i in (0, 1))
        x = torch.einsum("nhd,nkd->nhk", q[5 + a:5 + a + k.shape[0]].double(), k) / d ** 0.5
        hide = torch.arange(2 * bs, device="cuda") > last[a:a + 4096, None]
        want = torch.einsum("nhk,nkd->nhd", torch.softmax(x.masked_fill(hide[:, None], -torch.inf), -1), v)
        diff = out[5 + a:5 + a + k.shape[0]].double() - want
        assert float(diff.norm()) <= 1e-5 * float(want.norm()) and float(diff.abs().max()) <= 8e-5 * top


def test_attention_sequence_runs_report_bad_lengths():
    S = 65540
    pool = torch.zeros(1, 1, 2, 1, 4, 80, dtype=F16, device="cuda")
    q = torch.ones(S, 1, 80, device="cuda")
    for bad in (3, S - 1):
        pre = np.zeros(S)
        pre[bad] = 9                                          # past the table's one page
        f = new_flags()
        kv.cache_attention(q, pool, 0, i32(np.zeros((S, 1))), i32(np.arange(S + 1)), i32(pre), 1, 4, flags=f)
        assert int(f) == BAD_LENGTH


def test_attention_keeps_nothing_for_each_batch():
    """A server's calls differ in sequences and chunk lengths: the host's tables do not grow with them."""
    for d in (64, 96):
        seen = []
        for n in range(1, 9):
            b = Batch([(10 + n, n)] * n, 4, 2, d, 16, F16)
            b.run()
            seen.append(kv._workspace_bytes.cache_info().currsize)
        assert seen[-1] == seen[0]


@pytest.mark.parametrize("lens", [[20, 20], [16, 32], [20, 32]])
def test_fork_goes_on_after_it_ran_out_of_pages(lens):
    """Children without a page go on with their whole pages: counts stay those of the
    rows, in a call that continues some of them and in one that frees them all."""
    pool, table, _, refs = fork_case(lens, 4, 16, sum(-(-n // 16) for n in lens) + 2, shared=False)
    outside = refs.clone()
    for row, ln in zip(table.tolist(), lens):
        for page in row[:-(-ln // 16)]:
            outside[page] -= 1
    f = new_flags()

    def cut(t, n, s, r, written):
        """The lengths that go into the next call; the counts are those of the rows and the pages for their next tokens."""
        n = torch.where(s < 0, n // 16 * 16, n + written)
        want = outside.clone()
        for row, ln, slot in zip(t.tolist(), n.tolist(), s.tolist()):
            for page in {*row[:-(-ln // 16)], *([slot // 16] if slot >= 0 else [])}:
                want[page] += 1
        assert r.tolist() == want.tolist()
        return n

    t, n, s, r = kv.fork_pages(pool, table, i32(lens), i32([0, 0, 0, 1, 1]), refs, flags=f)
    assert int(f) == NO_PAGE and (s < 0).any() and (s >= 0).any()
    n = cut(t, n, s, r, 1)
    f.zero_()
    t, n, s, r = kv.fork_pages(pool, t, n, i32([int((s < 0).nonzero()[0]), int((s >= 0).nonzero()[0])]), r, flags=f)
    assert int(f) == 0 and (s >= 0).all()
    n = cut(t, n, s, r, 1)
    assert torch.equal(kv.fork_pages(pool, t, n, i32([]), r, flags=f)[3], outside) and int(f) == 0
