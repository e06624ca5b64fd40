"""Host side of the 16-bit cache: argument errors of the C entries (detected
before any launch), workspace sizes, compaction of the block pool on the host."""

import pytest
import torch

from kshipra_b200 import _lib
from kshipra_b200 import kv_cache as kv
from kshipra_b200.beam import BeamDecoder
from kshipra_b200.continuous import ContinuousEngine
from kshipra_b200.prefix_cache import PrefixCache

FAKE = 256          # never dereferenced: the arguments are checked before any launch


def test_sizes_need_no_device():
    h = _lib.lib()
    assert h.ksh_cache_attention_workspace_size(64, 32, 8, 128, 1) > 0
    assert h.ksh_cache_attention_workspace_size(1, 3, 2, 64, 4) == 0       # bad GQA ratio
    assert h.ksh_cache_attention_workspace_size(0, 4, 2, 64, 4) == 0
    assert h.ksh_fork_pages_scratch_ints(3, 5) >= 3 + 15
    assert h.ksh_compact_pages_scratch_ints(10) >= 11


def attention(h, **kw):
    a = dict(q=FAKE, total=4, hq=4, d=64, pool=FAKE, kind=1, nb=4, layers=1, layer=0, hkv=2, bs=16, bt=FAKE, maxb=2,
             qs=FAKE, pre=FAKE, seqs=1, maxq=4, tot=20, out=FAKE, ws=FAKE, wsb=1 << 30, flags=None)
    a.update(kw)
    return h.ksh_cache_attention(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(hq=3), dict(d=0), dict(kind=0), dict(kind=3), dict(nb=0), dict(layer=1), dict(layer=-1),
                                 dict(bs=0), dict(maxb=0), dict(seqs=-1), dict(total=-1), dict(maxq=-1), dict(q=None),
                                 dict(pool=None), dict(bt=None), dict(qs=None), dict(pre=None), dict(out=None),
                                 dict(total=1 << 31), dict(maxq=1 << 31)])
def test_attention_shape_errors(bad):
    assert attention(_lib.lib(), **bad) == -1


def test_attention_other_errors():
    h = _lib.lib()
    assert attention(h, d=320) == -4
    assert attention(h, ws=None) == -5
    assert attention(h, wsb=1) == -5
    assert attention(h, ws=FAKE + 8) == -2
    assert attention(h, seqs=0) == 0 and attention(h, total=0) == 0 and attention(h, maxq=0) == 0
    # past what the general kernel's grid can number
    assert attention(h, d=80, seqs=70000) == -4


def write(h, **kw):
    a = dict(qkv=FAKE, m=2, hq=4, hkv=2, d=64, pos=FAKE, slots=FAKE, cos=FAKE, sin=FAKE, maxpos=10, qn=None, kn=None, eps=1e-6,
             out=FAKE, pool=FAKE, kind=1, nb=4, layers=1, layer=0, bs=16, flags=None)
    a.update(kw)
    return h.ksh_rope_cache_write(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(m=-1), dict(hq=0), dict(hkv=0), dict(d=63), dict(d=0), dict(maxpos=0), dict(kind=5),
                                 dict(layer=2), dict(bs=0), dict(nb=0), dict(qkv=None), dict(pos=None), dict(slots=None),
                                 dict(cos=None), dict(sin=None), dict(out=None), dict(pool=None)])
def test_write_errors(bad):
    assert write(_lib.lib(), **bad) == -1
    assert write(_lib.lib(), m=0) == 0


def fork(h, **kw):
    a = dict(pool=FAKE, kind=1, nb=4, layers=1, hkv=2, bs=16, d=64, bt=FAKE, maxb=2, lens=FAKE, seqs=2, par=FAKE, n=3, ref=FAKE,
             nt=FAKE, nl=FAKE, slots=FAKE, nr=FAKE, scratch=FAKE, ints=1000, flags=None)
    a.update(kw)
    return h.ksh_fork_pages(*a.values(), None)


def compact(h, **kw):
    a = dict(pool=FAKE, kind=2, nb=4, layers=1, hkv=2, bs=16, d=64, bt=FAKE, entries=8, ref=FAKE, nt=FAKE, nr=FAKE, map=FAKE,
             used=FAKE, scratch=FAKE, ints=1000)
    a.update(kw)
    return h.ksh_compact_pages(*a.values(), None)


def test_pages_errors():
    h = _lib.lib()
    for bad in (dict(kind=9), dict(nb=0), dict(layers=0), dict(hkv=0), dict(bs=0), dict(d=0), dict(maxb=0), dict(seqs=-1),
                dict(n=-1), dict(pool=None), dict(bt=None), dict(lens=None), dict(ref=None), dict(nr=None), dict(par=None),
                dict(nt=None), dict(nl=None), dict(slots=None)):
        assert fork(h, **bad) == -1, bad
    assert fork(h, n=65536, ints=1 << 30) == -4
    assert fork(h, scratch=None) == -5 and fork(h, ints=5) == -5
    for bad in (dict(kind=9), dict(nb=0), dict(layers=0), dict(d=0), dict(entries=-1), dict(pool=None), dict(bt=None),
                dict(ref=None), dict(nt=None), dict(nr=None), dict(map=None), dict(used=None)):
        assert compact(h, **bad) == -1, bad
    assert compact(h, scratch=None) == -5 and compact(h, ints=3) == -5


def test_cpu_tensors_are_refused():
    pool = torch.zeros(4, 1, 2, 2, 16, 64, dtype=torch.float16)
    z = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: kv.cache_attention(torch.zeros(1, 4, 64), pool, 0, z.view(1, 1), z, z, 1, 1),
                 lambda: kv.rope_cache_write(torch.zeros(1, 512), pool, 0, z.long(), z.long(), torch.zeros(4, 32),
                                             torch.zeros(4, 32)),
                 lambda: kv.fork_pages(pool, z.view(1, 1), z, z, z),
                 lambda: kv.compact_pages(pool, z.view(1, 1), z)):
        with pytest.raises(_lib.KshipraLibraryError):
            call()


class _Model:
    tp_world, vocab_size = 1, 10


def test_beam_decoder_refusals():
    with pytest.raises(ValueError):
        BeamDecoder(_Model(), beams=0)
    with pytest.raises(ValueError):
        BeamDecoder(_Model(), beams=11)
    with pytest.raises(ValueError):
        BeamDecoder(_Model(), block_size=0)
    two = _Model()
    two.tp_world = 2
    with pytest.raises(ValueError):
        BeamDecoder(two)
    assert BeamDecoder(_Model()).generate([]) == []


def test_compaction_keeps_what_requests_and_the_tree_hold():
    """Blocks are named by what is written into them."""
    cache = PrefixCache(num_blocks=24, block_size=4, num_layers=2, num_kv_heads=1, head_dim=2, dtype=torch.float32)
    eng = ContinuousEngine(cache, 4, 64, 1.0, 0.05)
    pool = cache.allocator.pool
    reqs = [eng.add_request(list(range(100 * i, 100 * i + 9)), 3) for i in range(4)]
    tree_blocks = cache.allocate_blocks(2)
    node = cache.tree.insert(list(range(900, 908)), tree_blocks, 0, cache.tree.root)
    eng.schedule()
    for i, r in enumerate(reqs):
        for j, b in enumerate(r.block_table):
            pool[b] = 10.0 * i + j
    for j, b in enumerate(tree_blocks):
        pool[b] = 500.0 + j
    gone = eng.active_sequences.pop(reqs[1].req_id)
    for b in gone._own_blocks:
        cache.allocator.free(b)
    held = [r for r in reqs if r is not gone]
    used = sum(len(r.block_table) for r in held) + 2
    eng.compact()
    assert sorted(cache.allocator.free_blocks) == list(range(used, 24))
    assert cache.allocator.free_blocks[-1] == used               # the lowest goes first
    for i, r in enumerate(reqs):
        if r is gone:
            continue
        assert r._own_blocks == r.block_table and max(r.block_table) < used
        for j, b in enumerate(r.block_table):
            assert (pool[b] == 10.0 * i + j).all()
    assert all((pool[b] == 500.0 + j).all() for j, b in enumerate(node.block_ids))
    assert cache.tree.match(list(range(900, 908)))[0] == node.block_ids
    again = cache.compact()
    assert again == list(range(24))                               # nothing left to move


def test_compaction_of_empty_and_full_pools():
    cache = PrefixCache(num_blocks=5, block_size=4, num_layers=1, num_kv_heads=1, head_dim=2)
    assert cache.compact() == list(range(5))
    taken = cache.allocate_blocks(5)
    assert cache.compact() == list(range(5)) and cache.allocator.free_blocks == []
    cache.allocator.free(taken[2])
    to = cache.compact()
    assert to[4] == taken[2] if taken[2] != 4 else to == list(range(5))


def test_attention_workspace_size_depends_on_the_dimension_alone():
    size = _lib.lib().ksh_cache_attention_workspace_size
    for d in (64, 96, 128, 256):
        assert {size(s, h, k, d, n) for s in (1, 7, 70000) for h, k in ((1, 1), (32, 8), (256, 1)) for n in (0, 1, 5000)} == {size(1, 1, 1, d, 1)}
