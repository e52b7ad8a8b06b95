"""The decode step's operators under tensor parallelism (gloo, world 2): a
lockstep engine with an e4m3 cache, shared prefixes and filtered draws, and the
two-chunk decode pipeline against the plain forward."""

import os
from dataclasses import replace

import numpy as np
import pytest
import torch
import torch.multiprocessing as mp

from calfkit_amd.models.config import TINY

pytestmark = pytest.mark.dist


def _join(rank, world, port):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank), MASTER_ADDR="127.0.0.1",
                      MASTER_PORT=str(port))
    import calfkit_amd.parallel.pg as pg

    pg._DIST = None
    pg.init_distributed(backend="gloo", device_override="cpu")
    from calfkit_amd.models.llama import LlamaShard

    cfg = replace(TINY, heads=4, kv_heads=2, ffn=512)
    return LlamaShard(cfg, tp_rank=rank, tp_size=world, device="cpu")


def _leave():
    import torch.distributed as td

    td.barrier()
    td.destroy_process_group()


def _serving_worker(rank, world, port, q):
    model = _join(rank, world, port)
    from calfkit_amd import ops
    from calfkit_amd.engine import engine as engine_mod
    from calfkit_amd.engine.engine import GenRequest, InferenceEngine

    engine_mod.MIN_SHARED_BYTES = 0
    grouped = []
    inner = ops.build_prefix_groups

    def spy(*a, **kw):
        out = inner(*a, **kw)
        grouped.append(int((out[0] >= 0).sum()))
        return out

    ops.build_prefix_groups = spy
    engine = InferenceEngine(model, max_batch=4, use_graphs=False,
                             max_model_len=256, kv_dtype="fp8",
                             shared_prefix=True)
    if rank == 0:
        prefix = [1] + [7 + (i * 37) % 400 for i in range(130)]

        def serve(**kw):
            futs = [engine.submit(GenRequest(prompt_ids=prefix + [20 + i],
                                             max_new_tokens=9, **kw))
                    for i in range(3)]
            return [f.result(120).token_ids for f in futs]

        serve()  # the prefix's pages are there for all that follow
        outs = (serve(temperature=0.8, seed=3, top_p=0.5, top_k=1),
                serve(temperature=0.8, seed=3, top_p=0.9, min_p=0.01))
        engine.stop()
        q.put((rank, outs, max(grouped)))
    else:
        engine.follow()
        q.put((rank, None, max(grouped)))
    _leave()


def _run(worker, port):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=worker, args=(r, 2, port, q))
             for r in range(2)]
    for p in procs:
        p.start()
    got = sorted((q.get(timeout=180) for _ in procs), key=lambda g: g[0])
    for p in procs:
        p.join(timeout=120)
        assert p.exitcode == 0
    return got


def test_lockstep_engine_with_all_of_them():
    (_, outs, lead), (_, _, follow) = _run(_serving_worker, 29541)
    assert all(len(o) == 9 for out in outs for o in out)
    assert lead == follow == 3  # every rank groups the same rows


def _overlap_worker(rank, world, port, q):
    model = _join(rank, world, port)
    from calfkit_amd import ops
    from calfkit_amd.engine.kvcache import KVCache

    out = []
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        kv = KVCache(layers=model.cfg.layers, kv_heads=model.hkv,
                     head_dim=model.dh, num_pages=16, device="cpu",
                     dtype=dtype)
        scales = (list(zip(kv.kscale, kv.vscale)) if kv.kscale else None)
        g = torch.Generator().manual_seed(5)
        rows = torch.arange(16 * 64, dtype=torch.int32)
        for layer in range(model.cfg.layers):
            k, v = (torch.randn(rows.numel(), model.hkv, model.dh,
                                generator=g).to(torch.bfloat16)
                    for _ in range(2))
            if scales:
                ops.kv_write_fp8(kv.kcache[layer], kv.vcache[layer],
                                 *scales[layer], k, v, rows)
            else:
                ops.kv_write(kv.kcache[layer], kv.vcache[layer], k, v, rows)
        B = 4
        lens = torch.tensor([70, 90, 66, 100], dtype=torch.int32)
        table = torch.zeros(B, 4, dtype=torch.int32)
        table[:, 0] = 3
        table[:, 1] = torch.arange(B) + 5
        slots = (table[:, 1] * 64 + lens - 1 - 64).to(torch.int32)
        prefix = (torch.tensor([0, 0, -1, 0], dtype=torch.int32),
                  torch.tensor([64], dtype=torch.int32))
        torch.manual_seed(3)
        tokens = torch.randint(16, model.cfg.vocab_size, (B,))
        for overlap in ("0", "1"):
            os.environ["CALF_TP_OVERLAP"] = overlap
            out.append(model.forward(
                tokens, lens - 1, kv.kcache, kv.vcache, slots,
                page_table=table, seq_lens=lens, kv_scales=scales,
                prefix=prefix).float())
    q.put((rank, out, None))
    _leave()


def test_two_chunk_pipeline_matches_the_plain_forward():
    (_, out, _), _ = _run(_overlap_worker, 29543)
    for plain, lap in (out[:2], out[2:]):
        # as for the pipeline over the bf16 cache: the same sums in chunks
        assert torch.allclose(plain, lap, atol=1e-3, rtol=1e-3)


def _sliced(model, full, rank, world):
    """The shard's weights from one whole model's."""
    hq, hkv, dh, f = full.hq, full.hkv, full.dh, full.ffn_s

    def part(t, dim=0):
        return t.chunk(world, dim)[rank].contiguous()

    model.embed, model.lm_head = full.embed, full.lm_head
    for lw, fl in zip(model.layers, full.layers):
        heads = fl.wqkv.split([hq * dh, hkv * dh, hkv * dh])
        lw.wqkv = torch.cat([part(h) for h in heads])
        lw.wo = part(fl.wo, 1)
        lw.wgateup = torch.cat([part(h) for h in fl.wgateup.split([f, f])])
        lw.wdown = part(fl.wdown, 1)
    return model


def _drive(model, filters):
    """Prefill, prefill with prefix hits, decode to the end, in the same order
    on every rank.  -> (logits of every draw, tokens of every request)"""
    from concurrent.futures import Future

    from calfkit_amd import ops
    from calfkit_amd.engine.engine import GenRequest, InferenceEngine, _Seq

    eng = InferenceEngine(model, max_batch=4, use_graphs=False,
                          max_model_len=256, kv_dtype="fp8",
                          shared_prefix=True)
    prefix = [1] + [7 + (i * 37) % 400 for i in range(130)]
    seqs = [_Seq(i + 1, GenRequest(prompt_ids=prefix + [20 + i],
                                   max_new_tokens=9, ignore_eos=True,
                                   seed=40 + i, **f), Future())
            for i, f in enumerate(filters)]
    logits, inner = [], ops.sample
    # as arrays: a tensor in a queue belongs to the process that sent it
    ops.sample = lambda out, x, *a, **k: (
        logits.append(x.float().numpy().copy()), inner(out, x, *a, **k))[1]
    try:
        eng._prefill_batch(seqs[:1])
        eng._prefill_batch(seqs[1:])
        grouped = []
        while eng._running:
            eng._decode_step()
            grouped.append(int((eng._group >= 0).sum()))
    finally:
        ops.sample = inner
    assert max(grouped) == len(seqs)
    return logits, [s.result.token_ids for s in seqs]


def _values_worker(rank, world, port, q):
    shard = _join(rank, world, port)
    from calfkit_amd.engine import engine as engine_mod
    from calfkit_amd.models.llama import LlamaShard

    engine_mod.MIN_SHARED_BYTES = 0
    full = LlamaShard(shard.cfg, device="cpu")
    shard = _sliced(shard, full, rank, world)
    out = []
    for f in ([{}] * 3, [dict(temperature=0.8, top_p=0.9, min_p=0.01),
                         dict(temperature=1.0, top_p=0.5, top_k=40),
                         dict(temperature=0.7, min_p=0.02)]):
        out.append(_drive(shard, f))
    q.put((rank, out, _drive(full, [{}] * 3) if rank == 0 else None))
    _leave()


def test_sharded_engine_draws_the_tokens_of_every_rank_and_of_one():
    """Greedy and filtered requests over an e4m3 cache with shared prefixes:
    both ranks draw the same tokens, and the logits are those of the unsharded
    model."""
    (_, a, whole), (_, b, _) = _run(_values_worker, 29545)
    for (la, ta), (lb, tb) in zip(a, b):
        assert ta == tb and all(len(t) == 9 for t in ta)
        assert all((x == y).all() for x, y in zip(la, lb))
    # one rank rounds each of a layer's two projections once, two ranks round
    # both parts and their sum: 4 roundings of 2^-8 between them, over two
    # layers 16, 2^-4 if none cancels; rows stored in e4m3 that fall to another
    # code (2^-4 and less, where such a rounding tips them) double that
    bound = 2 ** -3
    (got, tokens), (want, alone) = a[0], whole
    assert len(got) == len(want)
    # draws: the first request's, the others', then the steps of all three
    rows = [[0], [1, 2]] + [[0, 1, 2]] * (len(got) - 2)
    same, compared = [True] * 3, 0
    step = [0, 0, 0]
    for x, y, members in zip(got, want, rows):
        for i, r in enumerate(members):
            if not same[r] or step[r] >= 9:
                continue
            size = np.linalg.norm(y[i])
            assert np.linalg.norm(x[i] - y[i]) <= bound * size
            t = tokens[r][step[r]]
            # the largest logit of one is within both errors of the other's
            assert y[i].max() - y[i][t] <= 2 * bound * size
            same[r] = t == alone[r][step[r]]
            step[r] += 1
            compared += 1
    assert compared >= 3
