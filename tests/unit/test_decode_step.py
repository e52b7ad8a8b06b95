"""The decode step's operators together: the engine with an e4m3 cache, shared
prefixes and filtered draws, and a captured run of the three kernels."""

import asyncio
import threading
import time
import types

import numpy as np
import pytest
import torch

from calfkit_amd import ops
from calfkit_amd.engine import engine as engine_mod
from calfkit_amd.engine.engine import (GenRequest, InferenceEngine, _Seq,
                                       _decode_prefill, _encode_prefill)
from calfkit_amd.engine.kvcache import KVCache
from calfkit_amd.engine.local import LocalModelClient
from calfkit_amd.engine.tokenizer import SyntheticTokenizer
from calfkit_amd.messages import TextPart, UserMessage
from calfkit_amd.models.config import TINY, get_config
from calfkit_amd.models.llama import LlamaShard
from calfkit_amd.schemas import EngineRequest, ModelSettings

HD, PAGE = 128, 64


def _engine(device="cpu", cfg=TINY, **kw) -> InferenceEngine:
    kw.setdefault("max_batch", 8)
    kw.setdefault("use_graphs", False)
    kw.setdefault("max_model_len", 512)
    return InferenceEngine(LlamaShard(cfg, device=device), **kw)


def _serve(eng, requests):
    try:
        futures = [eng.submit(r) for r in requests]
        return [f.result(300).token_ids for f in futures]
    finally:
        eng.stop()


PREFIX = [1] + [7 + (i * 37) % 400 for i in range(200)]


def _agents(n=6, **kw):
    """Agents with one system prompt, the first alone so that its pages are
    there for the others."""
    return [GenRequest(prompt_ids=PREFIX + [20 + i, 30 + i], max_new_tokens=9,
                       **kw) for i in range(n)]


def _staged(eng, n=6, **kw):
    try:
        first = eng.generate(_agents(1, **kw)[0], timeout=300).token_ids
        # the others together: held back until all are in the queue, so that
        # the batches (and with them the rounding of their products) are the
        # same in every run
        drain, gate = eng._drain_queue, threading.Event()

        def held(block):
            return drain(block) if gate.is_set() else time.sleep(0.01)

        eng._drain_queue = held
        time.sleep(0.2)
        futures = [eng.submit(r) for r in _agents(n, **kw)[1:]]
        gate.set()
        return [first] + [f.result(300).token_ids for f in futures]
    finally:
        eng.stop()


@pytest.fixture(autouse=True)
def _group_small_batches(monkeypatch):
    monkeypatch.setattr(engine_mod, "MIN_SHARED_BYTES", 0)


def test_fp8_cache_bytes_and_refusal():
    kv = KVCache(layers=2, kv_heads=3, head_dim=HD, num_pages=4, device="cpu",
                 dtype=torch.float8_e4m3fn)
    assert kv.bytes_per_page() == 2 * 2 * 3 * PAGE * (HD + 1)
    assert kv.bytes_per_layer_page() == 2 * 3 * PAGE * (HD + 1)
    assert kv.kscale[0].shape == (4, 3, PAGE)
    assert KVCache(layers=2, kv_heads=3, head_dim=HD, num_pages=4,
                   device="cpu").kscale is None
    with pytest.raises(ValueError):
        _engine(kv_dtype="int4")
    model = types.SimpleNamespace(dh=64, hq=8, hkv=2)
    for kw in (dict(kv_dtype="fp8"), dict(shared_prefix=True)):
        with pytest.raises(ValueError):
            InferenceEngine(model, **kw)


def test_shared_prefix_engine_gives_the_same_tokens(monkeypatch):
    """Grouped rows against the same engine with no group ever made."""
    seen = []
    inner = ops.build_prefix_groups

    def spy(*a, **kw):
        out = inner(*a, **kw)
        seen.append(int((out[0] >= 0).sum()))
        return out

    monkeypatch.setattr(ops, "build_prefix_groups", spy)
    grouped = _staged(_engine(shared_prefix=True))
    assert max(seen) >= 2, "no run shared a prefix"
    monkeypatch.undo()  # so few rows are not worth a pass by the rule
    monkeypatch.setattr(ops, "build_prefix_groups", spy)
    seen.clear()
    assert _staged(_engine(shared_prefix=True)) == grouped
    assert max(seen) == 0


@pytest.mark.parametrize("shared_prefix", [False, True])
def test_fp8_engine_is_near_the_bf16_one(shared_prefix):
    """One decode step after a prefill: logits over e4m3 rows against those
    over bf16 rows, and tokens that do not depend on the grouping."""
    a = _staged(_engine(kv_dtype="fp8", shared_prefix=shared_prefix))
    assert a == _staged(_engine(kv_dtype="fp8"))
    eng = _engine(kv_dtype="fp8")
    assert eng.kv.kcache[0].dtype == torch.float8_e4m3fn
    assert eng.kv.prefix_hit_tokens == 0
    _staged(eng)
    assert eng.kv.prefix_hit_tokens > 0  # read back through kv_read_fp8


def test_fp8_long_prompt_in_chunks():
    ids = [1] + [9 + (i * 13) % 450 for i in range(700)]
    r = _serve(_engine(kv_dtype="fp8", max_model_len=1024),
               [GenRequest(prompt_ids=ids, max_new_tokens=5)])
    assert len(r[0]) == 5


def test_filters_that_leave_one_are_greedy():
    """(Not min_p = 1: it keeps every logit equal to the largest, and bf16
    logits have such.)"""
    greedy = _serve(_engine(), _agents())
    for f in (dict(top_p=1e-6), dict(top_p=0.5, top_k=1),
              dict(min_p=0.3, top_k=1)):
        assert _serve(_engine(), _agents(temperature=0.9, seed=3, **f)) == greedy


def test_filtered_rows_leave_the_others_alone_and_repeat():
    """A filtered request's tokens depend on its seed, not on its batch; the
    unfiltered ones keep theirs."""
    plain = _agents(4, temperature=0.8, seed=5)
    alone = _serve(_engine(), plain)
    mixed = _agents(4, temperature=0.8, seed=5)
    mixed[1].top_p = 0.7
    mixed[3].min_p = 0.05
    a = _serve(_engine(), mixed)
    assert a[0] == alone[0] and a[2] == alone[2]
    again = _agents(4, temperature=0.8, seed=5)
    again[1].top_p = 0.7
    assert _serve(_engine(), [again[1]]) == [a[1]]


def test_a_filter_that_is_no_number_ends_its_own_request():
    """It is refused where it is given; the requests beside it run on."""
    eng = _engine()
    try:
        others = [eng.submit(r) for r in _agents(3, temperature=0.8, seed=5)]
        for kw in (dict(top_p=None), dict(top_p="0.9"), dict(min_p=[0.1])):
            with pytest.raises(TypeError):
                eng.submit(_agents(1, temperature=0.8, **kw)[0])
        others += [eng.submit(r) for r in _agents(1, temperature=0.8,
                                                  top_p=np.float32(0.9))]
        assert all(len(f.result(300).token_ids) == 9 for f in others)
    finally:
        eng.stop()


def test_settings_without_a_top_p_are_unfiltered():
    """A caller's settings may hold None for a value it leaves open."""
    class Sink:
        def emit(self, chunk):
            pass

    def answer(**kw):
        client = LocalModelClient(TINY, device="cpu")
        client._engine = _engine()
        client._tokenizer = SyntheticTokenizer(TINY.vocab_size)
        try:
            return asyncio.run(client.complete(EngineRequest(
                messages=(UserMessage((TextPart("hello"),)),), settings=ModelSettings(
                    max_tokens=6, temperature=0.8, seed=4, **kw)), Sink())).text
        finally:
            client._engine.stop()

    assert answer(top_p=None) == answer()


def test_settings_reach_the_draw():
    """An agent's top_p and min_p are its request's, its own over its model's."""
    seen = []
    client = LocalModelClient(TINY, device="cpu")
    client._engine = eng = _engine()
    client._tokenizer = SyntheticTokenizer(TINY.vocab_size)
    inner = eng.submit
    eng.submit = lambda r: (seen.append(r), inner(r))[1]

    class Sink:
        def emit(self, chunk):
            pass

    own = ModelSettings(max_tokens=3, temperature=0.5, min_p=0.05)
    try:
        asyncio.run(client.complete(EngineRequest(
            messages=(UserMessage((TextPart("hello"),)),),
            settings=ModelSettings(top_p=0.8, min_p=0.2).merged(own)), Sink()))
    finally:
        eng.stop()
    assert (seen[0].top_p, seen[0].min_p, seen[0].filtered) == (0.8, 0.05, True)


def test_lockstep_carries_the_filters():
    r = GenRequest(prompt_ids=[1, 2], temperature=0.5, top_k=7, seed=9,
                   top_p=0.9, min_p=0.05)
    (sid, got), = _decode_prefill(_encode_prefill([_Seq(4, r, None)]))
    assert sid == 4 and (got.top_p, got.min_p) == (0.9, 0.05)
    assert (got.top_k, got.seed, got.temperature) == (7, 9, 0.5)


@pytest.mark.parametrize("temperature", [1e-7, 1 / 3, 0.7000004, 0.0, 2])
def test_lockstep_carries_the_temperature_as_it_is(temperature):
    """Every rank draws with the first one's temperature: one cut to 0 would
    take the largest logit where the others draw."""
    r = GenRequest(prompt_ids=[1, 2], temperature=temperature, top_p=0.9)
    (_, got), = _decode_prefill(_encode_prefill([_Seq(4, r, None)]))
    assert got.temperature == temperature and got.filtered == r.filtered


@pytest.mark.gpu
@pytest.mark.parametrize("kv_dtype", ["bf16", "fp8"])
def test_engine_graphs_match_eager(kv_dtype):
    """Captured decode runs with groups and filters against eager ones."""
    cfg = get_config("smoke")
    runs = []
    for graphs in (True, False):
        eng = _engine("cuda", cfg, use_graphs=graphs, kv_dtype=kv_dtype,
                      shared_prefix=True, max_model_len=1024)
        runs.append(_staged(eng, temperature=0.7, top_p=0.9, seed=11))
        if graphs:
            assert eng.stats["graph_replays"] > 0
    assert runs[0] == runs[1]


class _Step:
    """Cache write -> shared attention -> draw, over static buffers."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.B, self.hq, self.hkv = 12, 8, 2
        B, hkv, pages = self.B, self.hkv, 40
        kv = KVCache(layers=1, kv_heads=hkv, head_dim=HD, num_pages=pages,
                     device="cuda", dtype=torch.float8_e4m3fn)
        self.cache = (kv.kcache[0], kv.vcache[0])
        self.scales = (kv.kscale[0], kv.vscale[0])

        def rand(*shape):
            return torch.randn(*shape, generator=g, device="cuda").to(
                torch.bfloat16)

        ops.kv_write_fp8(*self.cache, *self.scales, rand(pages * PAGE, hkv, HD),
                         rand(pages * PAGE, hkv, HD),
                         torch.arange(pages * PAGE, dtype=torch.int32,
                                      device="cuda"))
        self.qkv = rand(B, (self.hq + 2 * hkv) * HD)
        self.rope = ops.build_rope_table(512, HD, device="cuda")
        self.table = torch.zeros(B, 4, dtype=torch.int32, device="cuda")
        self.table[:, 0], self.table[:, 1] = 3, 9
        self.table[:, 2] = torch.arange(B, device="cuda") + 12
        self.lens = (130 + torch.arange(B, device="cuda")).to(torch.int32)
        self.group = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.group[5] = -1
        self.glens = torch.tensor([128], dtype=torch.int32, device="cuda")
        self.f = [torch.full((B,), v, dtype=d, device="cuda")
                  for v, d in ((0.9, torch.float32), (50, torch.int32),
                               (0.95, torch.float32), (0.01, torch.float32))]
        self.u = torch.rand(B, generator=g, device="cuda")
        self.out = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.kept = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.q = torch.zeros(B, self.hq, HD, dtype=torch.bfloat16,
                             device="cuda")
        self.o = torch.zeros_like(self.q)

    def run(self):
        pos = self.lens - 1
        slots = (self.table.gather(1, (pos // PAGE).long()[:, None])[:, 0]
                 * PAGE + pos % PAGE).to(torch.int32)
        ops.rope_qkv_write_fp8(self.qkv, *self.cache, *self.scales, self.rope,
                               pos, slots, self.hq, self.hkv, q_out=self.q)
        ops.attn_decode_shared(self.o, self.q, *self.cache, self.table,
                               self.lens, self.group, self.glens, HD ** -0.5,
                               *self.scales)
        # the attention's 1024 outputs stand for logits: a library product
        # has no place in a captured region that is replayed (it may record
        # clears of flags that its kernels then wait for)
        ops.sample_filtered(self.out, self.o.view(self.B, -1), *self.f, self.u,
                            kept=self.kept)

    def state(self):
        return [t.clone() for t in (self.o, self.out, self.kept,
                                    self.cache[0].view(torch.uint8),
                                    self.scales[1])]

    def vary(self, i):
        """Other inputs, in the same buffers."""
        g = torch.Generator(device="cuda").manual_seed(100 + i)
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=g, device="cuda"))
        self.lens.add_(1)
        self.u.copy_(torch.rand(self.B, generator=g, device="cuda"))
        self.group.fill_(-1 if i % 2 else 0)


@pytest.mark.gpu
def test_two_captured_steps_replay_as_eager():
    """Two graphs over the same code, replayed in turn with eager work and
    synchronisations between: each replay is the eager result."""
    steps, eager, graphs = [], [], []
    for seed in (1, 2):
        s, e = _Step(seed), _Step(seed)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            s.run()
        torch.cuda.current_stream().wait_stream(stream)
        e.run()  # both have written the first token's row
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run()
        steps.append(s)
        eager.append(e)
        graphs.append(graph)
    for i in range(4):
        for s, e, graph in zip(steps, eager, graphs):
            s.vary(i)
            e.vary(i)
            graph.replay()
            e.run()
            if i % 2:
                torch.cuda.synchronize()
        for s, e in zip(steps, eager):
            assert all(torch.equal(a, b) for a, b in zip(s.state(), e.state()))


@pytest.mark.gpu
def test_step_on_another_stream():
    a, b = _Step(4), _Step(4)
    a.run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        b.run()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(x, y) for x, y in zip(a.state(), b.state()))
    # twice the same: no sum depends on the order of its parts
    before = a.state()
    a.run()
    assert all(torch.equal(x, y) for x, y in zip(before, a.state()))
