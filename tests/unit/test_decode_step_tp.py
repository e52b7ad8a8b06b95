"""The decode step's operators under tensor parallelism (gloo, world 2): a
lockstep engine with an e4m3 cache, shared prefixes and filtered draws, and the
two-chunk decode pipeline against the plain forward."""

import os
from dataclasses import replace

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
