"""The inference engine: continuous batching + hipGraph-captured decode.

One engine per process (= per GPU rank).  Agent hops from every node hosted
by this worker funnel into the same engine, so concurrent agent turns batch
into one decode step — that is where whole-node agent turns/sec comes from.

Threading model: the engine owns a dedicated scheduler thread; the asyncio
agent plane submits requests through a thread-safe queue and gets
``concurrent.futures.Future``s back (bridged by LocalModelClient).

Decode runs (the hot loop):
  decode is data-independent except for the sampled token VALUES — slots,
  positions and sequence lengths all advance deterministically.  So the
  engine executes M consecutive decode steps per host visit: one hipGraph
  per (padded batch, M) contains M chained {forward -> sample -> feed the
  sampled ids back in on-device} steps over step-indexed static buffers,
  and the host syncs ONCE per run to read the M x B sampled ids.  Sequences
  that pass max_new/EOS mid-run overshoot by < M tokens; the extras are
  discarded and their KV pages truncated.
"""

from __future__ import annotations

import logging
import numbers
import queue
import struct
import threading
import time
from concurrent.futures import Future
from dataclasses import dataclass, field
from typing import Callable

import torch

from ..models.config import ModelConfig
from ..models.llama import LlamaShard
from .kvcache import KVCache, PAGE_SIZE

_log = logging.getLogger("calfkit.engine")

__all__ = ["GenRequest", "GenResult", "InferenceEngine"]

import os as _os

PREFILL_CHUNK = int(_os.environ.get("CALF_PREFILL_CHUNK", "512"))
#: token budget of one packed varlen prefill forward (the admission batch)
# r02 closing ABBA ladders: 12288 beat 8192 in both positions (239.8 vs
# 233.1 mean) and tied 16384 — bigger packed prefill batches feed the
# stream-K GEMMs better without hurting decode admission.
PREFILL_BUDGET = int(_os.environ.get("CALF_PREFILL_BUDGET", "12288"))
#: decode steps executed per host visit (graphs exist for each length).
#: 8 is the measured sweet spot: 16-step runs halve the per-visit host
#: cost but delay admission by a full run, and the running batch dips
#: enough to LOSE throughput end-to-end (233 -> 210 turns/s at 512)
RUN_STEPS = (8, 4, 2, 1)

#: prefix groups of one decode run (more share without being grouped)
MAX_PREFIX_GROUPS = 16
#: bytes of one layer's cache that groups save a step from being read, below
#: which rows run without them: a pass over prefixes and its join cost up to
#: 8 us.  Measured with cold caches, 32/8 heads, bf16, groups against none:
#: 67 MB (256 rows of 64 shared tokens) 97.9 against 90.0 us, 66 MB (64 of 256)
#: 31.8 / 32.5, 126 MB (16 of 2048) 23.8 / 25.3, 132 MB (64 of 512) 33.1 / 35.6,
#: 134 MB (256 of 128) 95.8 / 92.4, 252 MB (16 of 4096) 29.4 / 35.7, 264 MB (64
#: of 1024) 34.7 / 44.8; 16 pairs of 1024 (67 MB) 36.3 / 39.4, of 8192 162 / 187
MIN_SHARED_BYTES = 128 << 20

#: lockstep op channel opcodes (tensor-coded: the
#: pickled broadcast_object_list per visit becomes one fixed int64[2]
#: header broadcast, plus one int64 payload broadcast only for prefills)
OP_STOP, OP_DECODE, OP_PREFILL = 0, 1, 2


def _float_bits(x: float) -> int:
    return int.from_bytes(struct.pack("<d", x), "little", signed=True)


def _bits_float(i: int) -> float:
    return struct.unpack("<d", i.to_bytes(8, "little", signed=True))[0]


def _encode_prefill(seqs) -> list[int]:
    vals: list[int] = [len(seqs)]
    for s in seqs:
        r = s.request
        names = r.tool_names or []
        vals += [s.seq_id, r.max_new_tokens, _float_bits(r.temperature),
                 r.top_k, _float_bits(r.top_p), _float_bits(r.min_p), r.seed,
                 int(r.ignore_eos),
                 r.tool_trigger if r.tool_names else -1, r.tool_ncalls,
                 len(names)]
        vals += names
        vals.append(len(r.prompt_ids))
        vals += r.prompt_ids
    return vals


def _decode_prefill(vals: list[int]) -> list["GenRequest"]:
    reqs = []
    i = 1
    for _ in range(vals[0]):
        (sid, mx, temp, topk, topp, minp, seed, ig_eos, trig, ncalls,
         n_names) = vals[i:i + 11]
        i += 11
        names = vals[i:i + n_names]
        i += n_names
        n_ids = vals[i]
        i += 1
        ids = vals[i:i + n_ids]
        i += n_ids
        req = GenRequest(prompt_ids=list(ids), max_new_tokens=mx,
                         temperature=_bits_float(temp), top_k=topk,
                         top_p=_bits_float(topp), min_p=_bits_float(minp),
                         seed=seed,
                         ignore_eos=bool(ig_eos),
                         tool_names=list(names) if trig >= 0 else None,
                         tool_trigger=max(trig, 0), tool_ncalls=ncalls)
        reqs.append((sid, req))
    return reqs


_GOLDEN = 0x9E3779B97F4A7C15


def _row_key(seed: int, pos: int) -> int:
    """Per-(request, token-position) RNG key as a signed int64 (the sample
    kernel mix64's it with the vocab index)."""
    k = (seed * _GOLDEN + pos) & 0xFFFFFFFFFFFFFFFF
    return k - (1 << 64) if k >= (1 << 63) else k


def _uniforms(keys):
    """Row keys (uint64 array) -> the draws' random numbers in [0, 1), f32
    (24 bits of a 64-bit mix of the key)."""
    import numpy as np

    x = keys ^ (keys >> np.uint64(30))
    x = x * np.uint64(0xBF58476D1CE4E5B9)
    x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    x = x ^ (x >> np.uint64(31))
    return ((x >> np.uint64(40)).astype(np.float64) * 2.0 ** -24).astype(
        np.float32)


@dataclass
class GenRequest:
    prompt_ids: list[int]
    max_new_tokens: int = 64
    temperature: float = 0.0
    top_k: int = 0
    seed: int = 0
    ignore_eos: bool = True
    #: tool-call grammar plan: when tool_names is set the
    #: decode path runs grammar-constrained sampling — after tool_trigger
    #: generated tokens the model is steered into the TCALL <name> <args>
    #: TEND span, with the NAME genuinely sampled among these token ids.
    tool_names: "list[int] | None" = None
    tool_trigger: int = 0        # fire after this many generated tokens
    tool_ncalls: int = 1
    on_token: Callable[[int], None] | None = None
    #: batched delivery — called once per decode RUN with all tokens the
    #: run produced (and once with the prefill's first token).  When set,
    #: on_token is NOT called: one callback per host visit instead of one
    #: per token keeps the asyncio side from drowning in per-token tasks
    #: at large batch (profiles/r01_bench256_gaps.md).
    on_tokens: Callable[[list[int]], None] | None = None
    #: nucleus and relative-probability filters (1.0 and 0.0: off).  A request
    #: that uses either is drawn by ``ops.sample_filtered`` from one random
    #: number for each (seed, token position); the others by ``ops.sample``.
    top_p: float = 1.0
    min_p: float = 0.0

    @property
    def filtered(self) -> bool:
        return self.temperature > 0 and (self.top_p < 1 or self.min_p > 0)


@dataclass
class GenResult:
    token_ids: list[int] = field(default_factory=list)
    prompt_tokens: int = 0
    prefill_ms: float = 0.0
    decode_ms: float = 0.0
    finish_reason: str = "length"


@dataclass
class _Seq:
    seq_id: int
    request: GenRequest
    future: Future
    result: GenResult = field(default_factory=GenResult)
    last_token: int = 0
    new_tokens: int = 0
    #: host mirror of the device grammar state (transitions replayed over
    #: the sampled tokens after each run; gconsumed = tokens replayed)
    gstate: int = 0
    gconsumed: int = 0


@dataclass
class _PendingPrefill:
    """A prefill forward launched (possibly on the side stream) whose host
    finalization — first-token readback, bookkeeping, admission — is
    deferred until after the overlapped decode run."""
    seqs: list
    lens: list
    sampled: "torch.Tensor"  # [B] int32 on device
    t0: float


def _graph_batches() -> tuple:
    base = [1, 2, 4, 8, 16, 32, 64, 96, 128, 192, 256, 384, 512, 768, 1024]
    extra = _os.environ.get("CALF_EXTRA_GRAPH_BATCHES", "")
    for tok in extra.split(","):
        tok = tok.strip()
        if tok:
            base.append(int(tok))
    return tuple(sorted(set(base)))


class InferenceEngine:
    #: padded decode batch sizes that get their own captured graph
    #: (CALF_EXTRA_GRAPH_BATCHES adds sizes, e.g. "448,480" for finer
    #: padding near the serving point)
    GRAPH_BATCHES = _graph_batches()

    def __init__(self, model: LlamaShard, *, max_batch: int = 64,
                 kv_pages: int | None = None, use_graphs: bool | None = None,
                 max_model_len: int | None = None, kv_dtype: str = "bf16",
                 shared_prefix: bool = False):
        #: kv_dtype "fp8": the cache holds e4m3 codes with a power-of-two
        #: scale for each (token, head) — half the bytes, so twice the
        #: conversations a rank holds.  shared_prefix: decode attends a prefix
        #: that running sequences have in common (the same cached pages) once
        #: for all of them.
        if kv_dtype not in ("bf16", "fp8"):
            raise ValueError(f"kv_dtype must be 'bf16' or 'fp8': {kv_dtype!r}")
        if ((kv_dtype == "fp8" or shared_prefix)
                and (model.dh != 128 or model.hq > 16 * model.hkv)):
            raise ValueError(
                "kv_dtype='fp8' and shared_prefix need heads of 128 and up to "
                f"16 query heads a KV head, not {model.hq}/{model.hkv} heads "
                f"of {model.dh}")
        #: TP/EP>1 serving runs in lockstep: rank 0 schedules and broadcasts
        #: each action; ranks > 0 replay them via follow() — every rank then
        #: executes identical forwards (and RCCL collectives) in identical
        #: order, and identical seeds make the sampled tokens identical.
        self.tp_lockstep = (model.tp_size > 1
                            or getattr(model, "ep_size", 1) > 1)
        self.model = model
        self.cfg: ModelConfig = model.cfg
        self.device = model.device
        # round up to a graph batch size so padding never outgrows buffers
        for g in self.GRAPH_BATCHES:
            if max_batch <= g:
                max_batch = g
                break
        self.max_batch = max_batch
        self.max_model_len = max_model_len or self.cfg.max_seq
        self.on_gpu = self.device.type == "cuda"
        if use_graphs is None:
            # MoE decode is capturable through the grouped kernels
            # (ops/csrc/moe_gemm.hip): buckets are built device-side, so
            # there is no host sync.  The host-grouped fallback (no
            # extension) is not capturable — the capture try/except below
            # would catch it, but don't even try.
            from .. import ops as _ops
            # DECISION: TP/EP comm stays GRAPH-EXTERNAL.
            # RCCL-inside-hipGraph is unexercised on this stack, and the
            # TP-overlap pipeline (llama._forward_tp_overlap) already
            # multi-streams the collectives with event ordering — capture
            # would have to freeze that choreography.  tp/ep>1 therefore
            # decodes eager through the overlap pipeline; use_graphs=True
            # can still be forced explicitly for experiments.
            use_graphs = self.on_gpu and not self.tp_lockstep and (
                not self.cfg.is_moe
                or (_ops.have_extension()
                    and getattr(model, "ep_size", 1) == 1))
        self.use_graphs = use_graphs

        if kv_pages is None:
            # + max_batch: headroom for multi-step run overshoot (< RUN_STEPS
            # extra slots per sequence) and the padding dummy page
            kv_pages = ((max_batch * self.max_model_len + PAGE_SIZE - 1)
                        // PAGE_SIZE + 8 + max_batch)
        self.kv = KVCache(layers=self.cfg.layers, kv_heads=model.hkv,
                          head_dim=model.dh, num_pages=kv_pages,
                          device=self.device,
                          dtype=(torch.float8_e4m3fn if kv_dtype == "fp8"
                                 else torch.bfloat16))
        self._kv_scales = (list(zip(self.kv.kscale, self.kv.vscale))
                           if kv_dtype == "fp8" else None)
        # page-table width carries multi-step overshoot headroom: a sequence
        # at max_model_len batched with a longer-budget one blind-runs up to
        # RUN_STEPS[0]-1 extra slots before truncation
        from ..models.config import MAX_RUN_OVERSHOOT

        assert RUN_STEPS[0] <= MAX_RUN_OVERSHOOT
        self.max_pages = (self.max_model_len + RUN_STEPS[0]
                          + PAGE_SIZE - 1) // PAGE_SIZE

        # prefill scratch KV (contiguous [rows, hkv, dh] per layer).  The
        # packed varlen prefill with prefix-cache gathering lands the WHOLE
        # batch (pasts + new rows) here, so it must hold the full token
        # budget, not just one sequence
        scratch_rows = max(self.max_model_len, PREFILL_BUDGET)
        self._prefill_kv = [
            (torch.zeros(scratch_rows, model.hkv, model.dh,
                         dtype=model.dtype, device=self.device),
             torch.zeros(scratch_rows, model.hkv, model.dh,
                         dtype=model.dtype, device=self.device))
            for _ in range(self.cfg.layers)]

        # ---- static decode buffers (graph I/O); step-indexed for the
        # multi-step runs (MS = max run length)
        B = max_batch
        MS = RUN_STEPS[0]
        dev = self.device
        self._tokens = torch.zeros(B, dtype=torch.int64, device=dev)
        self._positions = torch.zeros(MS, B, dtype=torch.int32, device=dev)
        self._slots = torch.zeros(MS, B, dtype=torch.int32, device=dev)
        self._page_table = torch.zeros(B, self.max_pages, dtype=torch.int32,
                                       device=dev)
        self._seq_lens = torch.ones(MS, B, dtype=torch.int32, device=dev)
        self._temperature = torch.zeros(B, dtype=torch.float32, device=dev)
        self._topk = torch.zeros(B, dtype=torch.int32, device=dev)
        self._seeds = torch.zeros(MS, 2, dtype=torch.int64, device=dev)
        #: per-(step, row) RNG keys = request seed x token position, so a
        #: request's sampled tokens do not depend on batch composition
        self._row_seeds = torch.zeros(MS, B, dtype=torch.int64, device=dev)
        # filtered draws (top-p / min-p); a negative random number leaves the
        # row's token to ops.sample
        self._ftopk = torch.zeros(B, dtype=torch.int32, device=dev)
        self._topp = torch.ones(B, dtype=torch.float32, device=dev)
        self._minp = torch.zeros(B, dtype=torch.float32, device=dev)
        self._uniform = torch.full((MS, B), -1.0, dtype=torch.float32,
                                   device=dev)
        self._filters_set = False  # whether the buffers hold any
        # prefix groups of the running rows
        self.shared_prefix = shared_prefix
        self._group = torch.full((B,), -1, dtype=torch.int32, device=dev)
        self._group_lens = torch.zeros(MAX_PREFIX_GROUPS, dtype=torch.int32,
                                       device=dev)
        # tool-call grammar state (static graph I/O; trigger<0 = row off)
        from .. import ops as _gops

        self._gstate = torch.zeros(B, dtype=torch.int32, device=dev)
        self._gtrigger = torch.full((B,), -1, dtype=torch.int32, device=dev)
        self._gnames = torch.full((B, _gops.G_MAX_TOOLS), -1,
                                  dtype=torch.int32, device=dev)
        self._gncalls = torch.zeros(B, dtype=torch.int32, device=dev)
        self._sampled = torch.zeros(MS, B, dtype=torch.int32, device=dev)
        self._graphs: dict[tuple[int, int], torch.cuda.CUDAGraph] = {}
        #: one page sacrificed as the write target of padding rows
        self._dummy_page = self.kv.num_pages - 1
        self.kv._free.remove(self._dummy_page)

        # ---- prefill/decode overlap: waiting prompts prefill on a side
        # stream WHILE the decode graph replays (prefill is MFMA-bound,
        # decode HBM-bound — complementary).  Disjoint state: new seqs'
        # pages + prefill scratch vs running seqs' pages + decode buffers;
        # sampling gets its own candidate scratch so a concurrent decode
        # graph at the same batch size cannot race the shared one.
        self._s2 = torch.cuda.Stream(device=dev) if self.on_gpu else None
        self._prefill_cand = (torch.empty(B * 64 * 2, dtype=torch.float32,
                                          device=dev)
                              if self.on_gpu else None)
        self._pending: "_PendingPrefill | None" = None

        self._queue: "queue.Queue[_Seq | None]" = queue.Queue()
        self._running: list[_Seq] = []
        self._waiting: list[_Seq] = []
        self._next_id = 0
        self._step_counter = 0
        self._stats = {"decode_steps": 0, "decode_tokens": 0, "prefills": 0,
                       "decode_ms": 0.0, "prefill_ms": 0.0, "graph_replays": 0,
                       "idle_ms": 0.0}  # scheduler starved (no work queued)
        self._stop = threading.Event()
        self._thread = threading.Thread(target=self._loop, name="calfkit-engine",
                                        daemon=True)
        self._started = False
        self._lock = threading.Lock()

    # ------------------------------------------------------------- lifecycle
    def start(self) -> None:
        if not self._started:
            self._started = True
            self._thread.start()

    def stop(self) -> None:
        if self._started:
            self._stop.set()
            self._queue.put(None)
            self._thread.join(timeout=30)
            self._started = False
            if self.tp_lockstep:
                try:
                    self._op_bcast(OP_STOP)
                except Exception:
                    _log.exception("tp stop broadcast failed")

    @property
    def stats(self) -> dict:
        s = dict(self._stats)
        # KV/prefix-cache telemetry (observability parity with the step
        # ledger: the serving side of the mesh view)
        s["kv_pages_total"] = self.kv.num_pages
        s["kv_pages_free"] = self.kv.free_pages
        s["prefix_hit_tokens"] = self.kv.prefix_hit_tokens
        return s

    # ---------------------------------------------------------------- submit
    def submit(self, request: GenRequest) -> Future:
        """Thread-safe; returns a Future[GenResult]."""
        for name in ("top_p", "min_p"):  # here, where they end no one else's
            v = getattr(request, name)
            if not isinstance(v, numbers.Real):
                raise TypeError(f"{name} must be a number: {v!r}")
        self.start()
        fut: Future = Future()
        with self._lock:
            self._next_id += 1
            sid = self._next_id
        request.max_new_tokens = min(request.max_new_tokens,
                                     self.max_model_len - 1)
        if len(request.prompt_ids) + request.max_new_tokens > self.max_model_len:
            request.prompt_ids = request.prompt_ids[
                -(self.max_model_len - request.max_new_tokens):]
        self._queue.put(_Seq(seq_id=sid, request=request, future=fut))
        return fut

    def generate(self, request: GenRequest, timeout: float = 600.0) -> GenResult:
        return self.submit(request).result(timeout)

    # ----------------------------------------------------------- TP lockstep
    @property
    def _comm_dev(self) -> torch.device:
        from ..parallel import get_dist

        return self.device if get_dist().backend == "nccl" \
            else torch.device("cpu")

    def _op_bcast(self, opcode: int, payload: "list[int] | None" = None) -> None:
        if not self.tp_lockstep:
            return
        from ..parallel import broadcast_tensor

        dev = self._comm_dev
        n = len(payload) if payload else 0
        broadcast_tensor(torch.tensor([opcode, n], dtype=torch.int64,
                                      device=dev))
        if n:
            broadcast_tensor(torch.tensor(payload, dtype=torch.int64,
                                          device=dev))

    def _op_recv(self) -> "tuple[int, list[int] | None]":
        from ..parallel import broadcast_tensor

        dev = self._comm_dev
        hdr = torch.zeros(2, dtype=torch.int64, device=dev)
        broadcast_tensor(hdr)
        opcode, n = int(hdr[0]), int(hdr[1])
        vals = None
        if n:
            buf = torch.empty(n, dtype=torch.int64, device=dev)
            broadcast_tensor(buf)
            vals = buf.cpu().tolist()
        return opcode, vals

    def follow(self) -> None:
        """Follower loop for TP ranks > 0 (call instead of start())."""
        assert self.tp_lockstep
        if self.use_graphs:
            try:
                self._capture_graphs()
            except Exception:
                _log.exception("follower graph capture failed; eager")
                self.use_graphs = False
        while True:
            opcode, vals = self._op_recv()
            if opcode == OP_STOP:
                return
            if opcode == OP_PREFILL:
                if self._pending is not None:  # safety: rank 0 never does this
                    p, self._pending = self._pending, None
                    self._prefill_finalize(p)
                seqs = [_Seq(seq_id=sid, request=req, future=Future())
                        for sid, req in _decode_prefill(vals)]
                # mirror rank 0's deterministic overlap rule (lockstep state
                # is identical, so every rank takes the same branch)
                if self._overlap_ok(seqs):
                    with torch.cuda.stream(self._s2):
                        self._pending = self._prefill_launch(seqs)
                else:
                    self._prefill_batch(seqs)
            elif opcode == OP_DECODE:
                self._decode_step()
                if self._pending is not None:
                    p, self._pending = self._pending, None
                    self._prefill_finalize(p)

    # ------------------------------------------------------------------ loop
    def _loop(self) -> None:
        try:
            if self.use_graphs:
                self._capture_graphs()
        except Exception:
            _log.exception("hipGraph capture failed; falling back to eager")
            self.use_graphs = False
        while not self._stop.is_set():
            starved = not (self._running or self._waiting)
            if starved:
                t_idle = time.perf_counter()
            self._drain_queue(block=starved)
            if starved:
                self._stats["idle_ms"] += (time.perf_counter() - t_idle) * 1e3
            if self._stop.is_set():
                break
            try:
                # admit: pack waiting sequences into ONE varlen prefill
                # forward (token-budgeted); oversized prompts go chunked solo
                while self._waiting and len(self._running) < self.max_batch:
                    batch: list[_Seq] = []
                    budget = PREFILL_BUDGET
                    while (self._waiting and budget > 0
                           and len(self._running) + len(batch) < self.max_batch):
                        n = len(self._waiting[0].request.prompt_ids)
                        if n > PREFILL_BUDGET:
                            break  # long prompt: chunked solo below
                        if n > budget:
                            break
                        budget -= n
                        batch.append(self._waiting.pop(0))
                    if batch:
                        self._op_bcast(OP_PREFILL, _encode_prefill(batch))
                        if self._overlap_ok(batch):
                            # side-stream launch; the decode run below hides
                            # it — finalize (readback + admit) comes after
                            with torch.cuda.stream(self._s2):
                                self._pending = self._prefill_launch(batch)
                            break
                        self._prefill_batch(batch)
                    elif self._waiting:
                        solo = self._waiting.pop(0)
                        self._op_bcast(OP_PREFILL, _encode_prefill([solo]))
                        self._prefill_batch([solo])
                if self._running:
                    self._op_bcast(OP_DECODE)
                    self._decode_step()
                if self._pending is not None:
                    p, self._pending = self._pending, None
                    self._prefill_finalize(p)
            except Exception as e:
                _log.exception("engine step failed")
                pending = self._pending.seqs if self._pending else []
                self._pending = None
                for seq in self._running + self._waiting + pending:
                    if not seq.future.done():
                        seq.future.set_exception(e)
                    self.kv.release(seq.seq_id)
                self._running.clear()
                self._waiting.clear()

    def _drain_queue(self, block: bool) -> None:
        try:
            item = self._queue.get(timeout=0.05 if block else 0.0)
        except queue.Empty:
            return
        if item is not None:
            self._waiting.append(item)
        while True:
            try:
                item = self._queue.get_nowait()
            except queue.Empty:
                return
            if item is not None:
                self._waiting.append(item)

    # --------------------------------------------------------------- prefill
    def _prefill(self, seq: _Seq) -> None:
        t0 = time.perf_counter()
        ids = seq.request.prompt_ids
        n = len(ids)
        self.kv.open(seq.seq_id)
        model = self.model
        dev = self.device
        logits = None
        done = 0
        while done < n:
            chunk = ids[done:done + PREFILL_CHUNK]
            t = len(chunk)
            slots = self.kv.slots_for(seq.seq_id, t)
            tokens = torch.as_tensor(chunk, dtype=torch.int64, device=dev)
            positions = torch.arange(done, done + t, dtype=torch.int32,
                                     device=dev)
            slots_t = torch.as_tensor(slots, dtype=torch.int32, device=dev)
            logits = model.forward(
                tokens, positions, self.kv.kcache, self.kv.vcache, slots_t,
                prefill_scratch=self._prefill_kv, past_len=done,
                logits_rows=slice(t - 1, t), kv_scales=self._kv_scales)
            done += t
        assert logits is not None
        first = self._sample_host(logits, seq)
        if self.on_gpu:
            torch.cuda.synchronize(dev)
        seq.result.prompt_tokens = n
        seq.result.prefill_ms += (time.perf_counter() - t0) * 1e3
        self._stats["prefills"] += 1
        self._stats["prefill_ms"] += seq.result.prefill_ms
        self._emit_token(seq, first)
        self._emit_batch(seq, [first])
        if not self._finish_if_done(seq):
            self._running.append(seq)

    def _overlap_ok(self, seqs: list["_Seq"]) -> bool:
        """Prefill rides the side stream iff there is a decode run to hide
        it behind and the batch is not the chunked-solo long-prompt path.

        TP/EP lockstep engines never overlap: prefill and decode both issue
        RCCL collectives, and two streams' collectives interleaving
        differently across ranks is a classic deadlock."""
        import os

        # Default OFF: at the batch-256 operating point the A/B measured a
        # wash (the aggregate sits at the HBM roofline — see
        # profiles/r01_bench256_gaps.md), and overlapped admission shifts
        # decode batch shapes, whose library-GEMM tilings round
        # differently — greedy outputs then depend on arrival timing.
        # Opt in with CALF_PREFILL_OVERLAP=1 for latency-sensitive mixed
        # loads where hiding prefill behind decode matters more.
        return (self._s2 is not None and bool(self._running)
                and not self.tp_lockstep
                and os.environ.get("CALF_PREFILL_OVERLAP", "0") == "1"
                and not (len(seqs) == 1
                         and len(seqs[0].request.prompt_ids) > PREFILL_CHUNK))

    def _prefill_batch(self, seqs: list["_Seq"]) -> None:
        """Synchronous prefill: launch + finalize in one call."""
        if len(seqs) == 1 and len(seqs[0].request.prompt_ids) > PREFILL_CHUNK:
            return self._prefill(seqs[0])
        self._prefill_finalize(self._prefill_launch(seqs))

    def _prefill_launch(self, seqs: list["_Seq"]) -> _PendingPrefill:
        """Pack every waiting prompt into ONE varlen prefill forward and
        enqueue it (forward + first-token sampling) WITHOUT a host sync.

        Prefix-cached prompts prefill only their uncached SUFFIX: the cached
        pages are gathered into the contiguous scratch as the per-sequence
        past, and the new rows scatter into their packed positions.
        """
        if self.on_gpu:  # rocprofv3-visible phase marker (roctx via nvtx shim)
            torch.cuda.nvtx.range_push(f"calfkit.prefill[{len(seqs)}]")
        t0 = time.perf_counter()
        model = self.model
        dev = self.device
        cached: list[int] = []
        suffixes: list[list[int]] = []
        for s in seqs:
            c = self.kv.match_prefix(s.seq_id, s.request.prompt_ids)
            cached.append(c)
            suffixes.append(s.request.prompt_ids[c:])
        lens = [len(sx) for sx in suffixes]
        ids: list[int] = []
        positions: list[int] = []
        slots: list[int] = []
        q_starts_l = [0]
        kv_starts_l = [0]
        write_index: list[int] = []
        for s, sx, c in zip(seqs, suffixes, cached):
            ids.extend(sx)
            positions.extend(range(c, c + len(sx)))
            slots.extend(self.kv.slots_for(s.seq_id, len(sx)))
            write_index.extend(range(kv_starts_l[-1] + c,
                                     kv_starts_l[-1] + c + len(sx)))
            q_starts_l.append(q_starts_l[-1] + len(sx))
            kv_starts_l.append(kv_starts_l[-1] + c + len(sx))
        kv_total = kv_starts_l[-1]
        any_cached = any(cached)
        from .. import ops
        from ..models.llama import PrefillPlan

        if any_cached:
            self._gather_past(seqs, cached, kv_starts_l)
        q_starts = torch.as_tensor(q_starts_l, dtype=torch.int32).to(dev)
        kv_starts = torch.as_tensor(kv_starts_l, dtype=torch.int32).to(dev)
        plan = PrefillPlan(
            scratch=self._prefill_kv,
            block_map=ops.build_prefill_blocks(lens).to(dev),
            q_starts=q_starts,
            kv_starts=kv_starts,
            past_lens=torch.as_tensor(cached, dtype=torch.int32).to(dev),
            kv_write_start=0,
            kv_total=kv_total,
            kv_in_qkv=not any_cached,
            kv_write_index=(torch.as_tensor(write_index,
                                            dtype=torch.int64).to(dev)
                            if any_cached else None))
        logits = model.forward(
            torch.as_tensor(ids, dtype=torch.int64).to(dev),
            torch.as_tensor(positions, dtype=torch.int32).to(dev),
            self.kv.kcache, self.kv.vcache,
            torch.as_tensor(slots, dtype=torch.int32).to(dev),
            prefill_plan=plan,
            logits_rows=(q_starts[1:].long() - 1),
            kv_scales=self._kv_scales)
        for s in seqs:
            self.kv.register_prefix(s.seq_id, s.request.prompt_ids)
        sampled = self._sample_launch(logits, seqs)
        if self.on_gpu:
            torch.cuda.nvtx.range_pop()
        return _PendingPrefill(seqs=seqs, lens=lens, sampled=sampled, t0=t0)

    def _prefill_finalize(self, p: _PendingPrefill) -> None:
        """Host side of a launched prefill: read back first tokens, account,
        emit, admit to the running batch.  Under overlap this runs after
        the decode replay, so ``prefill_ms`` measures launch→finalize wall
        (it overstates GPU prefill time when overlapped — that is the
        point)."""
        if self._s2 is not None:
            self._s2.synchronize()  # no-op when launched on the default stream
        firsts = [int(t) for t in p.sampled.cpu()]
        if self.on_gpu:
            torch.cuda.synchronize(self.device)
        ms = (time.perf_counter() - p.t0) * 1e3
        self._stats["prefills"] += len(p.seqs)
        self._stats["prefill_ms"] += ms
        total_new = sum(p.lens)
        for s, n, tok in zip(p.seqs, p.lens, firsts):
            s.result.prompt_tokens = len(s.request.prompt_ids)
            s.result.prefill_ms += ms * n / max(1, total_new)  # by share
            self._emit_token(s, tok)
            self._emit_batch(s, [tok])
            if not self._finish_if_done(s):
                self._running.append(s)

    def _gather_past(self, seqs, cached, kv_starts_l) -> None:
        """Copy cached pages into the prefill scratch — ONE indexed gather +
        scatter per layer tensor.  (The per-sequence loop this replaced
        issued layers x seqs x 2 small torch ops; at 32 layers x 256
        sequences that was the dominant host gap in the batch-256 bench —
        see profiles/r01_bench256_gaps.md.)"""
        from .kvcache import PAGE_SIZE as PG

        pages_l: list[int] = []
        rows_l: list[int] = []
        for s, c, start in zip(seqs, cached, kv_starts_l[:-1]):
            if c == 0:
                continue
            pages_l.extend(self.kv._slots[s.seq_id].pages[: c // PG])
            rows_l.extend(range(start, start + c))
        if not pages_l:
            return
        dev = self.device
        if self._kv_scales is not None:
            # scratch row -> cache slot; rows still to be written: none
            slots = torch.full((kv_starts_l[-1],), -1, dtype=torch.int32)
            slots[torch.as_tensor(rows_l)] = (
                torch.as_tensor(pages_l, dtype=torch.int32)[:, None] * PG
                + torch.arange(PG, dtype=torch.int32)).view(-1)
            slots = slots.to(dev)
            from .. import ops

            for layer, (kbuf, vbuf) in enumerate(self._prefill_kv):
                ops.kv_read_fp8(kbuf[:slots.numel()], vbuf[:slots.numel()],
                                self.kv.kcache[layer], self.kv.vcache[layer],
                                *self._kv_scales[layer], slots)
            return
        pages = torch.as_tensor(pages_l, dtype=torch.long, device=dev)
        rows = torch.as_tensor(rows_l, dtype=torch.long, device=dev)
        hkv, dh = self.model.hkv, self.model.dh
        for layer in range(self.cfg.layers):
            kbuf, vbuf = self._prefill_kv[layer]
            kc, vc = self.kv.kcache[layer], self.kv.vcache[layer]
            # [P, hkv, PG, dh] -> gathered [n*PG, hkv, dh] at scratch rows
            kbuf[rows] = kc[pages].permute(0, 2, 1, 3).reshape(-1, hkv, dh)
            vbuf[rows] = vc[pages].permute(0, 2, 1, 3).reshape(-1, hkv, dh)

    def _sample_launch(self, logits: torch.Tensor,
                       seqs: list["_Seq"]) -> torch.Tensor:
        """Enqueue first-token sampling; returns the device tensor (no
        sync).  Uses the engine's own candidate scratch so it can run on
        the side stream concurrently with a decode graph."""
        from .. import ops

        B = len(seqs)
        out = torch.zeros(B, dtype=torch.int32, device=logits.device)
        temp = torch.as_tensor([s.request.temperature for s in seqs],
                               dtype=torch.float32).to(logits.device)
        topks = [0 if s.request.filtered else s.request.top_k for s in seqs]
        topk = torch.as_tensor(topks, dtype=torch.int32).to(logits.device)
        seed = torch.as_tensor(
            [seqs[0].request.seed or seqs[0].seq_id, self._step_counter],
            dtype=torch.int64).to(logits.device)
        rks = torch.as_tensor(
            [_row_key(s.request.seed or s.seq_id, 0) for s in seqs],
            dtype=torch.int64).to(logits.device)
        if any(s.request.tool_names for s in seqs):
            self._grammar_prefill(logits, seqs)
        ops.sample(out, logits, temp, seed,
                   topk if any(topks) else None,
                   cand=self._prefill_cand, row_seeds=rks)
        self._filter_first(out, logits, temp, seqs)
        return out

    @staticmethod
    def _filter_first(out: torch.Tensor, logits: torch.Tensor,
                      temp: torch.Tensor, seqs: list["_Seq"]) -> None:
        """Draw the first token of the requests that filter; the other rows
        keep what ``ops.sample`` gave them."""
        if not any(s.request.filtered for s in seqs):
            return
        import numpy as np

        from .. import ops

        keys = np.array([_row_key(s.request.seed or s.seq_id, 0)
                         for s in seqs], dtype=np.int64).view(np.uint64)
        u = np.where([s.request.filtered for s in seqs], _uniforms(keys),
                     np.float32(-1))
        dev = logits.device

        def row(values, dtype):
            return torch.as_tensor(values, dtype=dtype).to(dev)

        ops.sample_filtered(
            out, logits, temp,
            row([s.request.top_k for s in seqs], torch.int32),
            row([s.request.top_p for s in seqs], torch.float32),
            row([s.request.min_p for s in seqs], torch.float32),
            torch.from_numpy(u.astype(np.float32)).to(dev))

    def _grammar_prefill(self, logits: torch.Tensor,
                         seqs: list["_Seq"]) -> None:
        """Grammar bias for the first generated token (fresh state; the
        'previous' token is the last prompt token, never a special)."""
        from .. import ops

        dev = logits.device
        B = len(seqs)
        trig = torch.full((B,), -1, dtype=torch.int32)
        names = torch.full((B, ops.G_MAX_TOOLS), -1, dtype=torch.int32)
        ncalls = torch.zeros(B, dtype=torch.int32)
        pos = torch.zeros(B, dtype=torch.int32)
        prev = torch.zeros(B, dtype=torch.int64)
        for b, s in enumerate(seqs):
            prev[b] = s.request.prompt_ids[-1]
            pos[b] = len(s.request.prompt_ids) - 1
            if s.request.tool_names:
                trig[b] = pos[b] + s.request.tool_trigger
                ncalls[b] = s.request.tool_ncalls
                ids = s.request.tool_names[:ops.G_MAX_TOOLS]
                names[b, :len(ids)] = torch.as_tensor(ids, dtype=torch.int32)
        gstate = torch.zeros(B, dtype=torch.int32, device=dev)
        ops.grammar_bias(logits, prev.to(dev), gstate, trig.to(dev),
                         names.to(dev), pos.to(dev), ncalls.to(dev))

    def _sample_host(self, logits: torch.Tensor, seq: _Seq) -> int:
        r = seq.request
        out = torch.zeros(1, dtype=torch.int32, device=logits.device)
        temp = torch.full((1,), r.temperature, device=logits.device)
        seed = torch.as_tensor([r.seed or seq.seq_id, self._step_counter],
                               dtype=torch.int64, device=logits.device)
        rks = torch.as_tensor([_row_key(r.seed or seq.seq_id, 0)],
                              dtype=torch.int64, device=logits.device)
        topk = torch.full((1,), r.top_k, dtype=torch.int32, device=logits.device)
        from .. import ops
        if r.tool_names:
            self._grammar_prefill(logits, [seq])
        ops.sample(out, logits, temp, seed,
                   topk if r.top_k and not r.filtered else None,
                   row_seeds=rks)
        self._filter_first(out, logits, temp, [seq])
        return int(out.item())

    # ---------------------------------------------------------------- decode
    def _pad_batch(self, b: int) -> int:
        for g in self.GRAPH_BATCHES:
            if b <= g:
                return min(g, self.max_batch)
        return self.max_batch

    def _run_len(self) -> int:
        """Steps per host visit: bounded by the shortest remaining budget
        (a finishing sequence overshoots < M tokens, which is cheaper than
        shrinking every run to the laggard, but never run an entire batch
        past its collective end)."""
        rem = max(s.request.max_new_tokens - s.new_tokens
                  for s in self._running)
        for m in RUN_STEPS:
            if m <= rem:
                return m
        return 1

    def _write_run_state(self, pad: int, M: int) -> None:
        """Assemble the run's device state host-side with numpy (the
        python-nested-list version cost several ms per run at batch 256 —
        one of the per-run host gaps in profiles/r01_bench256_gaps.md)."""
        import numpy as np

        B = len(self._running)
        tokens = np.zeros(pad, dtype=np.int64)
        slots = np.empty((M, pad), dtype=np.int32)
        lens = np.ones((M, pad), dtype=np.int32)
        pt = np.zeros((pad, self.max_pages), dtype=np.int32)
        base = np.empty(pad, dtype=np.int32)
        base[B:] = 0
        run_slots = np.empty((B, M), dtype=np.int32)
        temps = np.zeros(pad, dtype=np.float32)
        topks = np.zeros(pad, dtype=np.int32)
        for b, s in enumerate(self._running):
            tokens[b] = s.last_token
            base[b] = self.kv.length(s.seq_id)
            run_slots[b] = self.kv.slots_for(s.seq_id, M)
            pages = self.kv._slots[s.seq_id].pages
            pt[b, :len(pages)] = pages
            temps[b] = s.request.temperature
            topks[b] = 0 if s.request.filtered else s.request.top_k
        steps = np.arange(M, dtype=np.int32)
        positions = base[None, :] + steps[:, None]
        lens = positions + 1
        slots[:, :B] = run_slots.T
        # padding rows decode against the dummy page
        slots[:, B:] = (self._dummy_page * PAGE_SIZE + steps)[:, None]
        pt[B:, 0] = self._dummy_page
        lens[:, B:] = 1
        self._tokens[:pad].copy_(torch.from_numpy(tokens), non_blocking=True)
        self._positions[:M, :pad].copy_(torch.from_numpy(positions),
                                        non_blocking=True)
        self._slots[:M, :pad].copy_(torch.from_numpy(slots), non_blocking=True)
        self._seq_lens[:M, :pad].copy_(torch.from_numpy(lens),
                                       non_blocking=True)
        self._page_table[:pad].copy_(torch.from_numpy(pt), non_blocking=True)
        self._temperature[:pad].copy_(torch.from_numpy(temps),
                                      non_blocking=True)
        self._topk[:pad].copy_(torch.from_numpy(topks), non_blocking=True)
        base_seed = self._running[0].request.seed or 12345
        seeds = [[base_seed, self._step_counter + i + 1] for i in range(M)]
        self._seeds[:M].copy_(torch.as_tensor(seeds, dtype=torch.int64),
                              non_blocking=True)
        # tool-call grammar rows: replay the mirror over tokens the device
        # has consumed (all but the newest), then load the static buffers
        from .. import ops as gops

        gtrig = np.full(pad, -1, dtype=np.int32)
        gnames = np.full((pad, gops.G_MAX_TOOLS), -1, dtype=np.int32)
        gncalls = np.zeros(pad, dtype=np.int32)
        gstates = np.zeros(pad, dtype=np.int32)
        for b, s in enumerate(self._running):
            if not s.request.tool_names:
                continue
            toks = s.result.token_ids
            while s.gconsumed < len(toks) - 1:
                s.gstate = gops.grammar_transition(s.gstate, toks[s.gconsumed])
                s.gconsumed += 1
            gstates[b] = s.gstate
            gtrig[b] = len(s.request.prompt_ids) - 1 + s.request.tool_trigger
            gncalls[b] = s.request.tool_ncalls
            ids = s.request.tool_names[:gops.G_MAX_TOOLS]
            gnames[b, :len(ids)] = ids
        self._gstate[:pad].copy_(torch.from_numpy(gstates), non_blocking=True)
        self._gtrigger[:pad].copy_(torch.from_numpy(gtrig), non_blocking=True)
        self._gnames[:pad].copy_(torch.from_numpy(gnames), non_blocking=True)
        self._gncalls[:pad].copy_(torch.from_numpy(gncalls),
                                  non_blocking=True)
        # per-row RNG keys: seed x token position (batch-composition-free)
        bases = np.array([(s.request.seed or s.seq_id) for s in self._running]
                         + [0] * (pad - B), dtype=np.uint64)
        toks = np.array([s.new_tokens for s in self._running]
                        + [0] * (pad - B), dtype=np.uint64)
        rk = (bases[None, :] * np.uint64(_GOLDEN)
              + (toks[None, :] + steps.astype(np.uint64)[:, None]))
        self._row_seeds[:M, :pad].copy_(
            torch.from_numpy(rk.view(np.int64)), non_blocking=True)
        filtered = np.zeros(pad, dtype=bool)
        filtered[:B] = [s.request.filtered for s in self._running]
        if filtered.any() or self._filters_set:
            ftopk = np.zeros(pad, dtype=np.int32)
            topp = np.ones(pad, dtype=np.float32)
            minp = np.zeros(pad, dtype=np.float32)
            ftopk[:B] = [s.request.top_k for s in self._running]
            topp[:B] = [s.request.top_p for s in self._running]
            minp[:B] = [s.request.min_p for s in self._running]
            self._uniform.fill_(-1.0)  # rows of other batch sizes too
            u = np.where(filtered[None, :], _uniforms(rk), np.float32(-1))
            self._uniform[:M, :pad].copy_(torch.from_numpy(u),
                                          non_blocking=True)
            for buf, rows in ((self._ftopk, ftopk), (self._topp, topp),
                              (self._minp, minp)):
                buf[:pad].copy_(torch.from_numpy(rows), non_blocking=True)
            self._filters_set = bool(filtered.any())
        if self.shared_prefix:
            group, lens = gops.build_prefix_groups(
                pt[:B], base[:B], max_groups=MAX_PREFIX_GROUPS,
                min_saved=MIN_SHARED_BYTES // self.kv.bytes_per_layer_page())
            full = np.full(pad, -1, dtype=np.int32)
            full[:B] = group
            self._group[:pad].copy_(torch.from_numpy(full), non_blocking=True)
            self._group_lens.copy_(torch.from_numpy(lens), non_blocking=True)
        self._step_counter += M

    def _decode_run_gpu(self, pad: int, M: int) -> None:
        """The captured region: M chained {forward -> sample} steps."""
        from .. import ops

        model = self.model
        tokens = self._tokens[:pad]
        for i in range(M):
            logits = model.forward(
                tokens, self._positions[i, :pad], self.kv.kcache,
                self.kv.vcache, self._slots[i, :pad],
                page_table=self._page_table[:pad],
                seq_lens=self._seq_lens[i, :pad],
                kv_scales=self._kv_scales,
                prefix=((self._group[:pad], self._group_lens)
                        if self.shared_prefix else None))
            # tool-call grammar: transition per-row state on the previous
            # token and bias the logits (no-op for rows without a plan)
            ops.grammar_bias(logits, tokens, self._gstate[:pad],
                             self._gtrigger[:pad], self._gnames[:pad],
                             self._positions[i, :pad], self._gncalls[:pad])
            ops.sample(self._sampled[i, :pad], logits,
                       self._temperature[:pad], self._seeds[i],
                       self._topk[:pad], row_seeds=self._row_seeds[i, :pad])
            # rows that filter by top-p or min-p are drawn again from their
            # own logits; without any, every block leaves at once (2.4 us)
            ops.sample_filtered(self._sampled[i, :pad], logits,
                                self._temperature[:pad], self._ftopk[:pad],
                                self._topp[:pad], self._minp[:pad],
                                self._uniform[i, :pad])
            tokens = self._sampled[i, :pad].long()  # on-device feedback

    def _capture_graphs(self) -> None:
        """One hipGraph per (padded batch, run length), largest first."""
        torch.cuda.synchronize(self.device)
        for b in reversed([g for g in self.GRAPH_BATCHES if g <= self.max_batch]):
            # full-length runs for every pad; short tail runs (M < 8) only
            # for small pads — large-batch tails are rare and run eager
            run_lens = RUN_STEPS if b <= 32 else RUN_STEPS[:1]
            for m in run_lens:
                self._decode_run_gpu(b, m)  # warm up allocations
                torch.cuda.synchronize(self.device)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    self._decode_run_gpu(b, m)
                self._graphs[(b, m)] = g
        torch.cuda.synchronize(self.device)
        _log.info("captured %d decode graphs: %s", len(self._graphs),
                  sorted(self._graphs))

    def _decode_step(self) -> None:
        t0 = time.perf_counter()
        B = len(self._running)
        pad = self._pad_batch(B)
        M = self._run_len()
        if self.on_gpu:
            torch.cuda.nvtx.range_push(f"calfkit.decode[{B}x{M}]")
        self._write_run_state(pad, M)
        if self.use_graphs and (pad, M) in self._graphs:
            self._graphs[(pad, M)].replay()
            self._stats["graph_replays"] += 1
        else:
            self._decode_run_gpu(pad, M)
        sampled = self._sampled[:M, :B].cpu()  # the ONE sync per run
        if self.on_gpu:
            torch.cuda.nvtx.range_pop()
        dt = (time.perf_counter() - t0) * 1e3
        self._stats["decode_steps"] += M
        self._stats["decode_tokens"] += M * B
        self._stats["decode_ms"] += dt
        from ..utils.metrics import metrics  # no-op shim unless enabled

        metrics.engine_tokens.labels(self.cfg.name, "decode").inc(M * B)
        metrics.engine_batch.labels(self.cfg.name).set(B)
        still: list[_Seq] = []
        for b, seq in enumerate(self._running):
            seq.result.decode_ms += dt
            done = False
            emitted: list[int] = []
            for i in range(M):
                t = int(sampled[i, b])
                self._emit_token(seq, t)
                emitted.append(t)
                done = self._check_done(seq)
                if done:
                    overshoot = M - 1 - i
                    if overshoot > 0:  # drop the blind-run extras
                        self.kv.truncate(seq.seq_id,
                                         self.kv.length(seq.seq_id) - overshoot)
                    break
            self._emit_batch(seq, emitted)
            if done:
                self._finish(seq)
            else:
                still.append(seq)
        self._running = still

    # --------------------------------------------------------------- helpers
    def _emit_token(self, seq: _Seq, token: int) -> None:
        seq.last_token = token
        seq.new_tokens += 1
        seq.result.token_ids.append(token)
        if seq.request.on_tokens is not None:
            return  # batched delivery at the call site
        cb = seq.request.on_token
        if cb is not None:
            try:
                cb(token)
            except Exception:
                _log.exception("on_token callback failed")

    @staticmethod
    def _emit_batch(seq: _Seq, tokens: list[int]) -> None:
        cb = seq.request.on_tokens
        if cb is not None and tokens:
            try:
                cb(tokens)
            except Exception:
                _log.exception("on_tokens callback failed")

    def _check_done(self, seq: _Seq) -> bool:
        r = seq.request
        eos_hit = (not r.ignore_eos) and seq.last_token == self.cfg.eos_id
        if eos_hit:
            seq.result.finish_reason = "stop"
            return True
        if seq.new_tokens >= r.max_new_tokens:
            seq.result.finish_reason = "length"
            return True
        return False

    def _finish(self, seq: _Seq) -> None:
        self.kv.release(seq.seq_id)
        if not seq.future.done():
            seq.future.set_result(seq.result)

    def _finish_if_done(self, seq: _Seq) -> bool:
        if self._check_done(seq):
            self._finish(seq)
            return True
        return False
