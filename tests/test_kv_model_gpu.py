"""KshipraModel over a 16-bit cache, with norms of queries and keys, and the
decoders and engines on top, against a plain forward in 64 bits.

The plain model rounds K and V to the cache's type where the kernels do, so what
is left between the two is fp32 arithmetic: logits within the 1e-3 (of the largest)
that the framework's other model tests take.  Tokens are compared where the plain
model's best two logits are further apart than 2e-3 of the largest (twice
the bound); at closer calls a stream may take either and is left there.
"""

import threading
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from kshipra_b200 import kv_cache as kv
from kshipra_b200.beam import BeamDecoder
from kshipra_b200.config import QWEN25_05B, TINY_LLAMA, ModelConfig, truncated
from kshipra_b200.continuous import ContinuousEngine
from kshipra_b200.model import KshipraModel
from kshipra_b200.prefix_cache import PrefixCache
from kshipra_b200.speculative import SpeculativeDecoder
from kshipra_b200.weights import synthetic_state_dict

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
RTOL = 1e-3
WIDE = ModelConfig(name="wide-heads", arch="llama", hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, intermediate=512,
                   vocab=1024, rope_theta=10000.0, max_positions=2048)


class Plain:
    """The forward of a Llama / Qwen2 model in 64 bits over whole sequences."""

    def __init__(self, cfg, sd, dtype):
        self.c, self.dtype = cfg, dtype
        self.w = {k: v.cuda().double() for k, v in sd.items()}

    def norm(self, x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + self.c.rms_eps) * w

    def logits(self, tokens):
        """[n, vocab] of one sequence."""
        c, w = self.c, self.w
        n, d, h, hk = len(tokens), c.head_dim, c.heads, c.kv_heads
        inv = 1.0 / (c.rope_theta ** (torch.arange(0, d, 2).float() / d))
        ang = torch.einsum("i,j->ij", torch.arange(n).float(), inv)
        cos, sin = ang.cos().double().cuda()[:, None], ang.sin().double().cuda()[:, None]

        def turn(x):
            a, b = x[..., : d // 2], x[..., d // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        x = w["model.embed_tokens.weight"][torch.tensor(tokens).cuda()]
        hide = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for i in range(c.layers):
            p = f"model.layers.{i}."
            lin = lambda y, name: y @ w[p + name + ".weight"].T + w.get(p + name + ".bias", 0.0)  # noqa: E731
            y = self.norm(x, w[p + "input_layernorm.weight"])
            q, k, v = (lin(y, f"self_attn.{s}_proj").view(n, -1, d) for s in "qkv")
            if p + "self_attn.q_norm.weight" in w:
                q, k = self.norm(q, w[p + "self_attn.q_norm.weight"]), self.norm(k, w[p + "self_attn.k_norm.weight"])
            q, k = turn(q), turn(k).to(self.dtype).double()
            v = v.to(self.dtype).double()
            k, v = k.repeat_interleave(h // hk, 1), v.repeat_interleave(h // hk, 1)
            s = torch.einsum("qhd,khd->hqk", q, k) / d ** 0.5
            o = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(hide, -torch.inf), -1), v)
            x = x + lin(o.reshape(n, -1), "self_attn.o_proj")
            y = self.norm(x, w[p + "post_attention_layernorm.weight"])
            g = lin(y, "mlp.gate_proj")
            x = x + lin(g * torch.sigmoid(g) * lin(y, "mlp.up_proj"), "mlp.down_proj")
        x = self.norm(x, w["model.norm.weight"])
        return x @ w.get("lm_head.weight", w["model.embed_tokens.weight"]).T


def normed(cfg, sd, seed=5):
    g = torch.Generator().manual_seed(seed)
    sd = dict(sd)
    for i in range(cfg.layers):
        for k in ("q_norm", "k_norm"):
            sd[f"model.layers.{i}.self_attn.{k}.weight"] = 1.0 + 0.2 * torch.randn(cfg.head_dim, generator=g)
    return sd


def close_call(row):
    top = row.topk(2).values
    return float(top[0] - top[1]) <= 2 * RTOL * float(row.abs().max())


def same_stream(plain, prompt, toks):
    """The greedy stream up to the first close call."""
    logits = plain.logits(list(prompt) + list(toks[:-1]))[len(prompt) - 1:]
    for row, t in zip(logits, toks):
        if int(row.argmax()) != t:
            assert close_call(row)
            return
        if close_call(row):
            return


def prompt_of(n, vocab, seed=0):
    return [int(x) for x in np.random.RandomState(seed).randint(0, vocab, n)]


CASES = [(TINY_LLAMA, F16, False), (TINY_LLAMA, BF16, True), (TINY_LLAMA, F32, True), (WIDE, BF16, False), (WIDE, F16, True),
         (truncated(QWEN25_05B, 2), F16, False)]


@pytest.mark.parametrize("cfg,dtype,norm", CASES, ids=lambda x: getattr(x, "name", str(x)))
def test_forward_and_generate(cfg, dtype, norm):
    sd = synthetic_state_dict(cfg, seed=1)
    if norm:
        sd = normed(cfg, sd)
    km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=dtype)
    plain = Plain(cfg, sd, dtype)
    prompt = prompt_of(75, cfg.vocab)
    alloc = km.new_pool(8, 16)
    assert alloc.pool.dtype is dtype
    bt, at = [5, 2, 7, 0, 1, 3], 0
    want = plain.logits(prompt)
    for n in (40, 1, 34):                                   # chunks, one of a single token
        pos = list(range(at, at + n))
        got = km.forward(torch.tensor([prompt[at:at + n]]), torch.tensor([pos]), alloc.pool, bt,
                         [bt[p // 16] * 16 + p % 16 for p in pos], at)
        w = want[at:at + n]
        assert float((got[0].double() - w).abs().max() / w.abs().max()) < RTOL
        at += n
    toks = km.generate(prompt, max_new_tokens=12, block_size=16, prefill_chunk=32)
    assert toks == km.generate(prompt, 12, block_size=16, use_graph=False)
    assert toks == km.generate(prompt, 12, block_size=16)   # the captured graph again
    same_stream(plain, prompt, toks)


@pytest.mark.parametrize("scheme", ["int8", "int4"])
def test_quantized_generate_is_the_fp32_pools(scheme):
    """The same prompt with an fp32 cache: the logits differ by the cache's rounding alone."""
    cfg = TINY_LLAMA
    sd = synthetic_state_dict(cfg, seed=0)
    prompt = prompt_of(50, cfg.vocab, 3)
    rows = []
    for dtype in (F32, F16):
        km = KshipraModel(config=cfg, state_dict=sd, quantize=scheme, kv_dtype=dtype)
        pool = km.new_pool(4, 16).pool
        pos = list(range(50))
        rows.append(km.forward(torch.tensor([prompt]), torch.tensor([pos]), pool, [0, 1, 2, 3], pos, 0)[0].double())
    # K and V off by 2^-11 of their size move a score by at most 2^-11 of |q||k| / sqrt(d), here below 1
    assert float((rows[0] - rows[1]).abs().max() / rows[0].abs().max()) < 2 * 2.0 ** -11 * cfg.layers + RTOL


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_engine_batches_and_preemption(dtype):
    cfg = TINY_LLAMA
    sd = normed(cfg, synthetic_state_dict(cfg, seed=2))
    km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=dtype)
    plain = Plain(cfg, sd, dtype)
    cache = PrefixCache(num_blocks=60, block_size=16, num_layers=cfg.layers, num_kv_heads=cfg.kv_heads, head_dim=cfg.head_dim,
                        dtype=dtype, device=km.device)
    eng = ContinuousEngine(cache, 16, 64, 64.0, 1.0, model=km)
    shared = prompt_of(40, cfg.vocab, 9)
    prompts = [shared + prompt_of(n, cfg.vocab, n) for n in (3, 17, 30, 1, 60)]
    reqs = [eng.add_request(p, 8) for p in prompts]
    for i in range(60):
        if not eng.waiting_queue and not eng.active_sequences:
            break
        eng.step()
        if i == 3:                                          # between steps: a request leaves and comes back,
            eng._preempt(next(iter(eng.active_sequences.values())))
        if i in (2, 4, 6):                                  # and the pool is compacted
            eng.compact()
    assert all(len(r.generated_tokens) == 8 for r in reqs)
    for p, r in zip(prompts, reqs):
        same_stream(plain, p, r.generated_tokens)


def plain_beams(plain, prompt, beams, steps, eos=None):
    """Beam search that runs every beam's whole sequence anew; (beams, whether no choice was close)."""
    live, clear = [([], 0.0, False)], True
    for _ in range(steps):
        cand = []
        for toks, score, done in live:
            if done:
                cand.append((toks, score, True))
                continue
            logp = torch.log_softmax(plain.logits(list(prompt) + toks)[-1], 0)
            vals, idx = logp.topk(beams + 1)
            cand += [(toks + [int(t)], score + float(v), eos is not None and int(t) == eos) for v, t in zip(vals, idx)]
        cand.sort(key=lambda c: -c[1])
        if len(cand) > beams and cand[beams - 1][1] - cand[beams][1] < 0.02:
            clear = False
        live = cand[:beams]
        if all(d for _, _, d in live):
            break
    gaps = [a[1] - b[1] for a, b in zip(live, live[1:])]
    return live, clear and all(g > 0.02 for g in gaps)


@pytest.mark.parametrize("dtype,beams,block", [(F16, 4, 16), (BF16, 3, 4), (F32, 4, 8), (F16, 1, 16), (F16, 6, 1)])
def test_beam_search(dtype, beams, block):
    """Scores add up log probabilities of logits within RTOL of the largest; choices
    that the plain search finds within 0.02 of each other end the comparison."""
    cfg = TINY_LLAMA
    sd = synthetic_state_dict(cfg, seed=4)
    sd = {k: v * (6.0 if k == "lm_head.weight" else 1.0) for k, v in sd.items()}      # scores that stand apart
    km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=dtype)
    plain = Plain(cfg, sd, dtype)
    prompts = [prompt_of(n, cfg.vocab, n) for n in (37, 1, 16, 33)]
    got = BeamDecoder(km, beams=beams, block_size=block).generate(prompts, max_new_tokens=7, prefill_chunk=16)
    compared = 0
    for p, beams_of in zip(prompts, got):
        assert len(beams_of) == beams and all(len(t) == 7 for t, _ in beams_of)
        assert [s for _, s in beams_of] == sorted((s for _, s in beams_of), reverse=True)
        for toks, score in beams_of:                        # each beam's score is its sequence's
            rows = torch.log_softmax(plain.logits(list(p) + toks[:-1])[len(p) - 1:], 1)
            want = float(rows[torch.arange(7), torch.tensor(toks).cuda()].sum())
            assert abs(score - want) < 0.02
        want, clear = plain_beams(plain, p, beams, 7)
        if clear:
            compared += 1
            assert [t for t, _ in beams_of] == [t for t, _, _ in want]
    assert compared > 0
    if beams == 1:
        for p, beams_of in zip(prompts, got):
            same_stream(plain, p, beams_of[0][0])


def test_beam_search_ends_and_penalties():
    cfg = TINY_LLAMA
    sd = synthetic_state_dict(cfg, seed=4)
    sd = {k: v * (6.0 if k == "lm_head.weight" else 1.0) for k, v in sd.items()}
    km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=F16)
    plain = Plain(cfg, sd, F16)
    prompt = prompt_of(21, cfg.vocab, 2)
    free = BeamDecoder(km, beams=4).generate([prompt], 6)[0]
    eos = free[0][0][2]
    got = BeamDecoder(km, beams=4).generate([prompt], 6, eos_token_id=eos)[0]
    want, clear = plain_beams(plain, prompt, 4, 6, eos)
    for toks, score in got:
        assert eos not in toks[:-1]
        rows = torch.log_softmax(plain.logits(prompt + toks[:-1])[len(prompt) - 1:], 1)
        assert abs(score - float(rows[torch.arange(len(toks)), torch.tensor(toks).cuda()].sum())) < 0.02
    if clear:
        assert [t for t, _ in got] == [t for t, _, _ in want]
    mean = BeamDecoder(km, beams=4, length_penalty=1.0).generate([prompt], 6, eos_token_id=eos)[0]
    by = sorted(((s / len(t), t) for t, s in got), key=lambda x: -x[0])
    assert [t for t, _ in mean] == [t for _, t in by]


def test_operators_together():
    """Fork, write, attend, compact, attend again: what each beam sees stays the same."""
    bs, hq, hkv, d = 8, 4, 2, 64
    rs = np.random.RandomState(0)
    pool = torch.zeros((40, 1, 2, hkv, bs, d), dtype=BF16, device="cuda")
    cos, sin = (torch.randn(64, d // 2, device="cuda") for _ in range(2))
    refs = torch.zeros(40, dtype=torch.int32, device="cuda")
    tables = torch.zeros((1, 8), dtype=torch.int32, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    parents, seen = [0], [[]]                               # the rows each sequence should hold
    for step in range(20):
        tables, lens, slots, refs = kv.fork_pages(pool, tables, lens, torch.tensor(parents, dtype=torch.int32).cuda(), refs, flags)
        seen = [list(seen[p]) for p in parents]
        n = len(parents)
        qkv = torch.randn(n, (hq + 2 * hkv) * d, device="cuda")
        q = kv.rope_cache_write(qkv, pool, 0, lens.long(), slots, cos, sin, flags=flags)
        rows = qkv.view(n, hq + 2 * hkv, d)
        a, b = rows[:, hq:hq + hkv, :d // 2], rows[:, hq:hq + hkv, d // 2:]
        c, s = cos[step][None, None], sin[step][None, None]
        k = torch.cat([a * c - b * s, b * c + a * s], -1).to(BF16)
        for i in range(n):
            seen[i].append((k[i], rows[i, hq + hkv:].to(BF16)))
        if step in (7, 13):
            tables, refs, _, used = kv.compact_pages(pool, tables, refs)
            assert int(used) == int((refs > 0).sum()) and int(tables.max()) < int(used)
            pool[int(used):] = float("nan")
        qs = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        got = kv.cache_attention(q, pool, 0, tables, qs, lens, 1, step + 1, flags=flags)
        for i in range(n):
            kk = torch.stack([x for x, _ in seen[i]], 1).double().repeat_interleave(hq // hkv, 0)
            vv = torch.stack([x for _, x in seen[i]], 1).double().repeat_interleave(hq // hkv, 0)
            w = torch.softmax(torch.einsum("hd,hkd->hk", q[i].double(), kk) / d ** 0.5, -1)
            want = torch.einsum("hk,hkd->hd", w, vv)
            assert float((got[i].double() - want).norm()) <= 1e-5 * float(want.norm())
        lens = lens + 1
        parents = [int(x) for x in rs.randint(0, n, rs.randint(1, 5))]
    assert int(flags) == 0


def test_refusals():
    cfg = TINY_LLAMA
    sd = synthetic_state_dict(cfg, seed=0)
    with pytest.raises(ValueError):
        KshipraModel(config=cfg, state_dict=sd, kv_dtype=torch.float64)
    km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=F16)
    with pytest.raises(ValueError):
        SpeculativeDecoder(km)
    with pytest.raises(ValueError):
        BeamDecoder(km).generate([[1] * 2048], 2)
    with pytest.raises(ValueError):
        BeamDecoder(km).generate([[]], 2)
    with pytest.raises(ValueError):
        km.prefill([1, 2, 3], km.new_pool(1, 16).pool.double(), [0])
    bad = normed(cfg, sd)
    bad["model.layers.0.self_attn.q_norm.weight"] = torch.ones(7)
    with pytest.raises(ValueError):
        KshipraModel(config=cfg, state_dict=bad)


def test_beam_search_ends_early_among_several_prompts():
    """An ended beam competes with itself alone: against the plain search wherever no
    choice of it is close, and at least one such search has a beam that ends early."""
    cfg = TINY_LLAMA
    sd = synthetic_state_dict(cfg, seed=4)
    sd = {k: v * (6.0 if k == "lm_head.weight" else 1.0) for k, v in sd.items()}
    km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=F16)
    plain = Plain(cfg, sd, F16)
    beams = BeamDecoder(km, beams=3, block_size=4)
    compared = 0
    for n in (5, 12, 21, 30, 37, 44):
        prompt = prompt_of(n, cfg.vocab, n)
        eos = beams.generate([prompt], 5)[0][0][0][1]         # the best beam's second token ends it now
        got = beams.generate([prompt], 5, eos_token_id=eos)[0]
        want, clear = plain_beams(plain, prompt, 3, 5, eos)
        if clear:
            assert [t for t, _ in got] == [t for t, _, _ in want]
            compared += any(len(t) < 5 and t[-1] == eos for t, _ in got)
    assert compared > 0


class Ranks:
    """Ranks as threads that issue their kernels to one stream in turn: what a
    collective takes from the others is there once all have come to it on the host."""

    def __init__(self, n):
        self.n, self.meet, self.parts, self.me = n, threading.Barrier(n, timeout=60), [None] * n, threading.local()

    def run(self, fn):
        def rank(r):
            self.me.rank = r
            try:
                return fn(r)
            except BaseException:
                self.meet.abort()
                raise
        with ThreadPoolExecutor(self.n) as ex:
            return [f.result() for f in [ex.submit(rank, r) for r in range(self.n)]]

    def gather(self, t):
        self.parts[self.me.rank] = t.clone()
        self.meet.wait()
        parts = list(self.parts)
        self.meet.wait()
        return parts

    def all_reduce(self, t, group=None):
        t.copy_(torch.stack(self.gather(t)).sum(0))

    def all_gather_into_tensor(self, out, t, group=None):
        out.copy_(torch.stack(self.gather(t)))


@pytest.mark.parametrize("cfg,dtype,norm", [(TINY_LLAMA, F16, False), (TINY_LLAMA, BF16, True), (TINY_LLAMA, F32, True), (WIDE, F16, True)],
                         ids=lambda x: getattr(x, "name", str(x)))
def test_tensor_parallel_shards(cfg, dtype, norm, monkeypatch):
    """Shards over pools of each type, with norms of queries and keys: chunks and a
    single token give the whole model's logits."""
    monkeypatch.setenv("KSH_PEER_AR", "0")
    sd = synthetic_state_dict(cfg, seed=3)
    sd = normed(cfg, sd) if norm else sd
    ranks = Ranks(2)
    monkeypatch.setattr(torch.distributed, "all_reduce", ranks.all_reduce)
    monkeypatch.setattr(torch.distributed, "all_gather_into_tensor", ranks.all_gather_into_tensor)
    prompt = prompt_of(40, cfg.vocab, 1)

    def rank(r):
        km = KshipraModel(config=cfg, state_dict=sd, kv_dtype=dtype, tp=(r, 2, None))
        pool = km.new_pool(5, 8).pool
        assert pool.dtype == dtype and pool.shape[3] == cfg.kv_heads // 2
        rows, at = [], 0
        for n in (21, 18, 1):
            rows.append(km.forward(torch.tensor([prompt[at:at + n]]), torch.arange(at, at + n)[None], pool, [3, 0, 4, 1, 2],
                                   [[3, 0, 4, 1, 2][i // 8] * 8 + i % 8 for i in range(at, at + n)], at)[0])
            at += n
        return torch.cat(rows)

    got = ranks.run(rank)
    want = Plain(cfg, sd, dtype).logits(prompt)
    for x in got:
        assert float((x.double() - want).abs().max()) <= RTOL * float(want.abs().max())
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=["fp16", "bf16", "fp32"])
def test_prefix_cache_compacts_on_the_gpu_as_on_the_host(dtype):
    caches = [PrefixCache(num_blocks=50, block_size=4, num_layers=2, num_kv_heads=2, head_dim=64, dtype=dtype, device=torch.device(dev))
              for dev in ("cuda", "cpu")]
    rs = np.random.RandomState(0)
    data = torch.randn(caches[0].allocator.pool.shape, generator=torch.Generator().manual_seed(0)).to(dtype)
    drop = [int(b) for b in rs.permutation(30)[:17]]
    for c in caches:
        c.allocator.pool.copy_(data)
        held = c.allocate_blocks(30)
        c.node = c.tree.insert(list(range(12)), [b for b in held if held.index(b) not in drop][:3], 0, c.tree.root)
        for i in drop:
            c.allocator.free(held[i])
        c.before = set(held) - {held[i] for i in drop}
        c.blocks = list(c.node.block_ids)
        c.to = c.compact()
    gpu, cpu = caches
    assert gpu.to == cpu.to and gpu.to != list(range(50)) and gpu.allocator.free_blocks == cpu.allocator.free_blocks
    for c in caches:
        assert sorted(c.to[b] for b in c.before) == list(range(13))
        assert c.node.block_ids == [c.to[b] for b in c.blocks]
        for b in c.before:
            assert torch.equal(c.allocator.pool[c.to[b]].cpu(), data[b])


def test_drafted_trees_in_a_model_with_norms():
    """Trees over an fp32 pool with norms of queries and keys: the model's greedy streams."""
    cfg = TINY_LLAMA
    sd = normed(cfg, synthetic_state_dict(cfg, seed=6))
    km = KshipraModel(config=cfg, state_dict=sd)
    plain = Plain(cfg, sd, F32)
    a = prompt_of(11, cfg.vocab, 3)
    prompts = [a * 4, a, prompt_of(33, cfg.vocab, 4)]
    for p, toks in zip(prompts, SpeculativeDecoder(km).generate(prompts, 12)):
        assert len(toks) == 12
        same_stream(plain, p, toks)
