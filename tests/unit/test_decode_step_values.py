"""What an engine with an e4m3 cache computes, against an engine with a bf16
cache that is made to hold the same values: cache rows, logits and the scratch
rows of a prefix hit."""

from concurrent.futures import Future

import pytest
import torch

from calfkit_amd import ops
from calfkit_amd.engine import engine as engine_mod
from calfkit_amd.engine.engine import GenRequest, InferenceEngine, _Seq
from calfkit_amd.models.config import get_config
from calfkit_amd.models.llama import LlamaShard

PAGE = 64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _two_to(e):
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _rounded(x):
    """The values an e4m3 row with a power-of-two scale holds, in 64 bits."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(a, -127)
    for lift in (128, 64, 32, 16, 8, 4, 2, 1):
        e = torch.where(a > 448.0 * _two_to(e + lift - 1), e + lift, e)
    e = torch.where(a > 0, e, 0.0)
    y = x * _two_to(-e)
    octave = torch.frexp(y.abs().clamp_min(2.0 ** -6))[1] - 1
    y = torch.round(y * _two_to(3 - octave)) * _two_to(octave - 3)
    return y * _two_to(e)


def _held(kv, layer):
    """(K, V) of an e4m3 cache in 64 bits."""
    return [c[layer].float().double() * _two_to(s[layer].int() - 127).unsqueeze(-1)
            for c, s in ((kv.kcache, kv.kscale), (kv.vcache, kv.vscale))]


class _Pair:
    """One model behind an e4m3 and a bf16 engine that are given the same."""

    def __init__(self, device, monkeypatch, **kw):
        cfg = get_config("tiny" if device == "cpu" else "smoke")
        model = LlamaShard(cfg, device=device)
        self.e4m3, self.bf16 = self.engines = [
            InferenceEngine(model, max_batch=8, use_graphs=False,
                            max_model_len=1024, kv_dtype=t, **kw)
            for t in ("fp8", "bf16")]
        self.logits = []
        inner = ops.sample

        def spy(out, logits, *a, **k):
            self.logits.append(logits.float().cpu())
            return inner(out, logits, *a, **k)

        monkeypatch.setattr(ops, "sample", spy)

    def prefill(self, first_id, prompts):
        """Both engines' first-token logits."""
        self.logits.clear()
        for eng in self.engines:
            eng._prefill_batch([
                _Seq(first_id + i,
                     GenRequest(prompt_ids=list(p), max_new_tokens=9,
                                ignore_eos=True), Future())
                for i, p in enumerate(prompts)])
        return self.logits

    def rows(self, seq_id):
        """(pages, offsets) of a sequence's tokens, the same in both."""
        a, b = ([e.kv._slots[seq_id].pages, e.kv.length(seq_id)]
                for e in self.engines)
        assert a == b
        at = torch.arange(a[1])
        return torch.tensor(a[0])[at // PAGE], at % PAGE

    def check_rows(self, seq_ids):
        """Every token's row is the bf16 engine's, rounded."""
        for layer in range(self.e4m3.cfg.layers):
            held = _held(self.e4m3.kv, layer)
            for x, y in zip(held, (self.bf16.kv.kcache, self.bf16.kv.vcache)):
                for seq in seq_ids:
                    pages, at = self.rows(seq)
                    want = _rounded(y[layer][pages, :, at])
                    assert torch.equal(x[pages, :, at], want)
                    assert want.abs().sum() > 0

    def same_values(self):
        """The bf16 cache is given what the e4m3 one holds (bf16 has room)."""
        for layer in range(self.e4m3.cfg.layers):
            for x, y in zip(_held(self.e4m3.kv, layer),
                            (self.bf16.kv.kcache, self.bf16.kv.vcache)):
                y[layer].copy_(x)


PREFIX = [1] + [7 + (i * 37) % 400 for i in range(200)]


def test_e4m3_prefill_holds_the_bf16_rows_rounded(monkeypatch):
    """Fresh prompts, a prompt in chunks, then prompts whose first pages are
    read back: no layer, scale or row is another's.  A prompt's own rows are
    attended as bf16, so that nothing but the stored rows differs, and with the
    same past nothing differs at all."""
    p = _Pair("cpu", monkeypatch)
    a, b = p.prefill(1, [PREFIX + [20], PREFIX[:90], [1, 5, 9]])
    assert torch.equal(a, b)
    p.check_rows([1, 2, 3])
    long = [1] + [9 + (i * 13) % 450 for i in range(700)]
    assert len(long) > engine_mod.PREFILL_CHUNK
    a, b = p.prefill(4, [long])
    assert torch.equal(a, b)
    p.check_rows([4])
    # the second and third begin with pages that are there: 192 and 64 tokens
    p.same_values()
    hits = p.e4m3.kv.prefix_hit_tokens
    a, b = p.prefill(5, [[3, 4], PREFIX + [33, 34], PREFIX[:64] + [8] * 70])
    assert p.e4m3.kv.prefix_hit_tokens - hits == 192 + 64
    assert torch.equal(a, b)
    p.same_values()
    p.check_rows([5, 6, 7])


@pytest.mark.parametrize("device", DEVICES)
def test_e4m3_gather_past_reads_every_layers_rows(device, monkeypatch):
    """The scratch rows of a prefix hit are the cached ones, each in its layer
    and place; the rows of the suffixes are left alone."""
    p = _Pair(device, monkeypatch)
    eng = p.e4m3
    p.prefill(1, [PREFIX, [9] + PREFIX])
    prompts = [PREFIX[:130] + [8], [2, 3], [9] + PREFIX[:70]]
    seqs = [_Seq(10 + i, GenRequest(prompt_ids=x), Future())
            for i, x in enumerate(prompts)]
    cached = [eng.kv.match_prefix(s.seq_id, s.request.prompt_ids)
              for s in seqs]
    assert cached == [128, 0, 64]
    starts = [0]
    for x in prompts:
        starts.append(starts[-1] + len(x))
    for k, v in eng._prefill_kv:
        k.fill_(7.0)
        v.fill_(7.0)
    eng._gather_past(seqs, cached, starts)
    for layer, scratch in enumerate(eng._prefill_kv):
        for held, got in zip(_held(eng.kv, layer), scratch):
            left = torch.ones(got.shape[0], dtype=torch.bool)
            for s, c, at in zip(seqs, cached, starts):
                pages = eng.kv._slots[s.seq_id].pages[:c // PAGE]
                if c:
                    want = held[pages].transpose(1, 2).reshape(c, *got.shape[1:])
                    assert want.abs().sum() > 0
                    assert torch.equal(got[at:at + c].double(), want)
                    left[at:at + c] = False
            assert (got.cpu()[left] == 7.0).all()


def _step(eng):
    """One eager decode step's logits; (the run's own draws are not read)."""
    B = len(eng._running)
    eng._write_run_state(B, 1)
    return eng.model.forward(
        eng._tokens[:B], eng._positions[0, :B], eng.kv.kcache, eng.kv.vcache,
        eng._slots[0, :B], page_table=eng._page_table[:B],
        seq_lens=eng._seq_lens[0, :B], kv_scales=eng._kv_scales,
        prefix=((eng._group[:B], eng._group_lens)
                if eng.shared_prefix else None)).float().cpu()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shared", [False, True])
def test_e4m3_decode_step_gives_the_logits_of_its_values(device, shared,
                                                         monkeypatch):
    """One decode step over e4m3 rows against one over a bf16 cache with the
    same values, the new token's row rounded likewise."""
    monkeypatch.setattr(engine_mod, "MIN_SHARED_BYTES", 0)
    p = _Pair(device, monkeypatch, shared_prefix=shared)
    p.prefill(1, [PREFIX + [20]])
    p.prefill(2, [PREFIX + [21, 22], [1, 5, 9], PREFIX + [23]])
    assert len(p.e4m3._running) == 4
    for a, b in zip(p.e4m3._running, p.bf16._running):
        a.last_token = b.last_token = 11     # the draws may differ
    p.same_values()
    got = _step(p.e4m3)
    if shared:
        assert int((p.e4m3._group[:4] >= 0).sum()) == 3

    def rounding(inner, kc, slots):
        def write(*a):
            inner(*a)
            for cache in (a[kc], a[kc + 1]):
                s = a[slots].long()
                rows = cache[s // PAGE, :, s % PAGE]
                cache[s // PAGE, :, s % PAGE] = _rounded(rows).to(cache.dtype)

        return write

    monkeypatch.setattr(ops, "rope_qkv_write",
                        rounding(ops.rope_qkv_write, 1, 5))
    monkeypatch.setattr(ops, "rope_qkv_write_slab",
                        rounding(ops.rope_qkv_write_slab, 2, 6))
    if shared:
        # each row by itself: the grouping is not to matter
        monkeypatch.setattr(ops, "build_prefix_groups", lambda t, n, **kw: (
            -torch.ones(len(n), dtype=torch.int32).numpy(),
            torch.zeros(engine_mod.MAX_PREFIX_GROUPS,
                        dtype=torch.int32).numpy()))
    want = _step(p.bf16)
    # the values are the same: what differs is the order of 32-bit sums, and
    # with it the rounding of a layer's attention to bf16, by one step (2^-7) of
    # each value at most, as much in the next layer's
    layers = p.e4m3.cfg.layers
    err = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert (err <= layers * 2 ** -7).all(), err
