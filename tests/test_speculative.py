"""Host side of speculative decoding: drafts, argument errors of the C entries
(detected before any launch) and workspace sizes."""

import random

import pytest
import torch

from kshipra_b200 import _lib
from kshipra_b200 import speculative as sp
from kshipra_b200.speculative import PromptLookup

FAKE = 256          # never dereferenced: the arguments are checked before any launch


def walk(tokens, parents, node):
    out = []
    while node > 0:
        out.append(tokens[node])
        node = parents[node]
    return out[::-1]


def test_prompt_lookup_merges_continuations():
    toks, par = PromptLookup(ngram=2, depth=3, branches=3, max_nodes=8).propose(
        [1, 2, 9, 8, 1, 2, 9, 7, 1, 2])
    assert toks[0] == 2 and par[0] == -1
    assert all(0 <= p < i for i, p in enumerate(par) if i)
    paths = {tuple(walk(toks, par, i)) for i in range(1, len(toks))}
    assert {(9, 7, 1), (9, 8, 1)} <= paths
    # no child of a node twice
    assert len({(p, t) for p, t in zip(par, toks)}) == len(toks)


def test_prompt_lookup_limits():
    assert PromptLookup().propose([4]) == ([4], [-1])
    assert PromptLookup().propose([1, 2, 3]) == ([3], [-1])
    toks, par = PromptLookup(ngram=1, depth=50, branches=50, max_nodes=5).propose([7] * 40)
    assert len(toks) == 5 and par == [-1, 0, 1, 2, 3]
    for bad in (dict(ngram=0), dict(max_nodes=0), dict(max_nodes=257), dict(depth=-1)):
        with pytest.raises(ValueError):
            PromptLookup(**bad)


def test_workspace_size_needs_no_device():
    h = _lib.lib()
    assert h.ksh_tree_attention_workspace_size(64, 32, 8, 128, 16) > 0
    assert h.ksh_tree_attention_workspace_size(1, 3, 2, 64, 4) == 0        # bad GQA ratio
    assert h.ksh_tree_attention_workspace_size(0, 4, 2, 64, 4) == 0


def attention(h, **kw):
    a = dict(q=FAKE, total=4, hq=4, d=64, pool=FAKE, nb=4, layers=1, layer=0, hkv=2, bs=16, bt=FAKE,
             maxb=2, qs=FAKE, pre=FAKE, seqs=1, mask=FAKE, words=1, nodes=4, tot=20, out=FAKE, ws=FAKE,
             wsb=1 << 30, flags=None)
    a.update(kw)
    return h.ksh_tree_attention(*a.values(), None)


def test_argument_errors_are_reported_without_a_launch():
    h = _lib.lib()
    for kw, st in ((dict(hq=5), -1), (dict(layer=1), -1), (dict(bs=0), -1), (dict(q=None), -1),
                   (dict(mask=FAKE, words=0), -1), (dict(d=257), -4), (dict(nodes=257), -4),
                   (dict(words=5), -4), (dict(total=-1), -1), (dict(bs=1 << 31), -1),
                   (dict(nb=1 << 30), -4)):     # K/V rows numbered in 32 bits
        assert attention(h, **kw) == st, kw
    # nothing to do is no error
    for kw in (dict(seqs=0), dict(total=0), dict(nodes=0)):
        assert attention(h, **kw) == 0

    def tables(seqs=1, total=4, bs=16, ids=FAKE, start=FAKE, maxb=2, par=FAKE, words=1, qs=FAKE,
               bt=FAKE, pos=FAKE, mask=FAKE):
        return h.ksh_tree_tables(FAKE, FAKE, seqs, total, bs, ids, 2, start, maxb, par, words, qs, bt,
                                 pos, FAKE, mask, None, None)
    for kw, st in ((dict(seqs=0), -1), (dict(bs=0), -1), (dict(start=None), -1), (dict(maxb=0), -1),
                   (dict(words=5), -4), (dict(words=0), -1), (dict(mask=None), -1), (dict(pos=None), -1),
                   (dict(qs=None), -1)):
        assert tables(**kw) == st, kw

    def verify(seqs=1, nodes=4, vocab=10, tp=FAKE, ts=10, dp=None, ds=10, tt=None, u=FAKE, path=FAKE):
        return h.ksh_verify_tree(FAKE, FAKE, FAKE, seqs, 4, nodes, vocab, tp, ts, dp, ds, tt, u, FAKE,
                                 path, FAKE, FAKE, None, None)
    for kw, st in ((dict(seqs=0), -1), (dict(nodes=0), -1), (dict(nodes=257), -4), (dict(vocab=0), -1),
                   (dict(ts=9), -1), (dict(tp=None), -1), (dict(tt=FAKE), -1), (dict(u=None), -1),
                   (dict(dp=FAKE, ds=9), -1), (dict(tp=None, tt=FAKE, dp=FAKE), -1), (dict(path=None), -1)):
        assert verify(**kw) == st, kw

    assert h.ksh_target_probs(FAKE, 2, 10, 9, None, FAKE, 10, None) == -1
    assert h.ksh_target_probs(FAKE, 2, 0, 9, None, FAKE, 10, None) == -1
    assert h.ksh_target_probs(None, 2, 10, 10, None, FAKE, 10, None) == -1
    assert h.ksh_target_probs(None, 0, 10, 10, None, None, 10, None) == 0
    assert h.ksh_tree_commit(FAKE, 4, 1, 2, 16, 64, FAKE, 2, FAKE, 0, FAKE, 4, FAKE, None, None, None) == -1
    assert h.ksh_tree_commit(FAKE, 4, 1, 2, 16, 64, FAKE, 2, FAKE, 1, FAKE, 0, FAKE, None, None, None) == -1
    assert h.ksh_tree_commit(None, 4, 1, 2, 16, 64, FAKE, 2, FAKE, 1, FAKE, 4, FAKE, None, None, None) == -1


class On:
    """What the checks look at of a tensor on some device."""

    is_cuda = True

    def __init__(self, device, shape, dtype=torch.int32):
        self.t = torch.empty(shape, dtype=dtype)
        self.device_index = device

    def get_device(self):
        return self.device_index

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_tensors_of_one_call_are_on_one_device():
    ok = On(1, (4,))
    assert sp._need(ok, "x", torch.int32, 1) is ok and sp._need(ok, "x", torch.int32, 1, 1) is ok
    rows = On(1, (2, 3), torch.float32)
    assert sp._rows(rows, "x", 1) is rows and sp._flags(None, 1) is None
    assert sp._flags(ok, 1) == ok.data_ptr()
    for bad in (lambda: sp._need(ok, "x", torch.int32, 1, 0), lambda: sp._rows(rows, "x", 0),
                lambda: sp._flags(ok, 0),
                lambda: sp._flags(On(1, (1,), torch.int64), 1), lambda: sp._flags(On(1, (0,)), 1),
                # no launch follows: the first tensors differ
                lambda: sp.tree_tables(ok, On(0, (4,)), 4, 16, 4, 1, block_tables=On(1, (4, 1))),
                lambda: sp.tree_attention(On(0, (2, 2, 64), torch.float32), On(1, (1, 1, 2, 2, 16, 64), torch.float32),
                                          0, ok, ok, ok, None, 1, 1),
                lambda: sp.target_probs(rows, On(0, (2,), torch.float32)),
                lambda: sp.verify_tree(On(0, (4,), torch.int64), ok, ok, 2, target_tokens=ok),
                lambda: sp.commit_tree(On(0, (1, 1, 2, 2, 16, 64), torch.float32), On(1, (1, 1)), ok, ok, ok)):
        with pytest.raises(ValueError):
            bad()
    cpu = torch.zeros(4, dtype=torch.int32)
    for bad in (lambda: sp._need(cpu, "x", torch.int32, 1), lambda: sp._flags(cpu, 0),
                lambda: sp._rows(torch.zeros(2, 3), "x")):
        with pytest.raises(_lib.KshipraLibraryError):
            bad()


def test_rows_past_32_bit_element_numbers_are_refused():
    h = _lib.lib()
    for v in ((1 << 30) + 1, (1 << 31) - 1):
        assert h.ksh_target_probs(FAKE, 1, v, v, None, FAKE, v, None) == -4
        assert h.ksh_verify_tree(FAKE, FAKE, FAKE, 1, 4, 4, v, FAKE, v, None, 0, None, FAKE, FAKE, FAKE, FAKE,
                                 FAKE, None, None) == -4


def test_workspace_is_kept_by_what_may_still_use_it(monkeypatch):
    """A captured graph holds the buffer's address: no later call may replace the
    buffer, and a capture takes one of its own."""
    real, capturing = torch.empty, [False]
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: real(n, dtype=dtype))
    monkeypatch.setattr(sp, "_raw_stream", lambda idx: 7 + idx)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    size = {d: _lib.lib().ksh_tree_attention_workspace_size(4, 8, 2, d, 8) for d in (64, 80, 128)}
    assert size[80] < size[64] < size[128]
    dev, ws = torch.device("cuda", 0), sp.TreeWorkspace()
    first = ws.get(size[80], dev)
    assert ws.get(size[64], dev) is first and ws.get(size[128], dev) is first
    capturing[0] = True
    a, b = ws.get(size[64], dev), ws.get(size[128], dev)
    assert len({t.data_ptr() for t in (first, a, b)}) == 3
    assert a.numel() >= size[64] and b.numel() >= size[128]
    capturing[0] = False
    assert ws.get(size[128], dev) is first


def test_cut_keeps_the_nodes_down_to_a_depth():
    toks, par = [9, 1, 2, 3, 4, 5, 6], [-1, 0, 1, 0, 2, 3, 5]
    assert sp.cut_tree(toks, par, 3) == (toks, par)
    assert sp.cut_tree(toks, par, 2) == ([9, 1, 2, 3, 5], [-1, 0, 1, 0, 3])
    assert sp.cut_tree(toks, par, 1) == ([9, 1, 3], [-1, 0, 0])
    assert sp.cut_tree(toks, par, 0) == ([9], [-1])
    # a parent that is no earlier node stays one for the device to report
    assert sp.cut_tree([9, 1, 2, 3], [-1, 3, 0, 2], 1) == ([9, 1, 2], [-1, -1, 0])
    for depth in (1, 9):                        # arrays as well as lists
        a, b = sp.cut_tree(torch.tensor(toks).numpy(), torch.tensor(par).numpy(), depth)
        assert (a, b) == sp.cut_tree(toks, par, depth)
    for bad in (([], []), ([1, 2], [-1])):
        with pytest.raises(ValueError):
            sp.cut_tree(*bad, 1)


@pytest.mark.parametrize("ngram,depth,branches,nodes", [(3, 6, 3, 16), (1, 4, 9, 40), (4, 2, 1, 3), (2, 0, 3, 8),
                                                        (3, 5, 0, 8), (2, 7, 5, 1)])
def test_lookup_of_a_growing_sequence_is_the_scans(ngram, depth, branches, nodes):
    lookup = PromptLookup(ngram, depth, branches, nodes)
    for seed in range(6):
        r = random.Random(seed)
        tokens = [r.randrange(2 + seed) for _ in range(r.choice([1, 2, 9, 60]))]
        seq = lookup.sequence(tokens)
        for _ in range(25):
            assert seq.propose() == lookup.propose(tokens)
            new = [r.randrange(2 + seed) for _ in range(r.randrange(4))]
            tokens = tokens + new
            seq.extend(new)


def test_lookup_reads_what_it_drafts_not_the_history():
    class Counted(list):
        reads = 0

        def __getitem__(self, i):
            got = super().__getitem__(i)
            Counted.reads += len(got) if isinstance(i, slice) else 1
            return got

        def __iter__(self):
            Counted.reads += len(self)
            return super().__iter__()

    lookup = PromptLookup(ngram=3, depth=6, branches=3, max_nodes=16)
    for tokens in (list(range(30000)), [i % 997 for i in range(30000)], [5] * 30000):
        seq = lookup.sequence(tokens)
        seq.tokens = Counted(seq.tokens)
        for step in range(5):
            Counted.reads = 0
            seq.extend([7, 8])
            seq.propose()
            assert Counted.reads <= 2 * (1 + 2 + 3) + 6 + 1 + 3 * 6


def test_a_proposers_own_propose_is_called():
    class Mine(PromptLookup):
        def propose(self, tokens):
            return [tokens[-1], len(tokens)], [-1, 0]

    class Plain:
        max_nodes = 2

        def propose(self, tokens):
            tokens.append(99)                   # its own copy
            return [tokens[-2], len(tokens) - 1], [-1, 0]

    for proposer in (Mine(), Plain()):
        seq = sp.sequence_of(proposer, [4, 6])
        assert seq.propose() == ([6, 2], [-1, 0])
        seq.extend([3])
        assert seq.propose() == ([3, 3], [-1, 0])


def test_calls_run_on_their_tensors_device(monkeypatch):
    """From another current device the entry runs under the tensors' one, on its
    current stream."""
    now, log = [0], []

    class Under:
        def __init__(self, device):
            self.to = device.index

        def __enter__(self):
            self.was, now[0] = now[0], self.to

        def __exit__(self, *exc):
            now[0] = self.was

    class Entries:
        def ksh_some_entry(self, *args):
            log.append((now[0],) + args)
            return 0

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Under)
    monkeypatch.setattr(sp, "_raw_stream", lambda idx: 100 + idx)
    monkeypatch.setattr(sp._lib, "lib", Entries)
    for idx in (0, 3):
        sp._run(torch.device("cuda", idx), "ksh_some_entry", 5, None)
    assert log == [(0, 5, None, 100), (3, 5, None, 103)] and now == [0]
