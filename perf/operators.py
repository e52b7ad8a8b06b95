"""The decode-step operators and their plain forms, as cases to be measured.

Four operators of one decode step of a serving engine:

- ``write``:  rotate the packed QKV rows, quantise K and V to e4m3 with one
  power-of-two scale for each (token, KV head) as they go into the paged cache,
  and read the written rows back;
- ``decode``: single-token grouped-query attention over that quantised cache;
- ``shared``: the same attention for a batch whose rows share long prefixes,
  each prefix computed once for its whole group (bf16 or e4m3 cache);
- ``sample``: a token from temperature, top-k, top-p and min-p and one given
  random number for each row.

``run`` computes the plain forms with elementary torch operations, or, where
``own`` is true, calls ``calfkit_amd.ops``.
"""

import math

import torch

own = False

HD = 128      # head size of every configuration
PAGE = 64     # tokens of one cache page
DEV = "cuda"


def listed():
    return [
        # one agent's single new token, 8B heads: latency alone
        dict(name="write-1", kind="write", T=1, hq=32, hkv=8),
        # a full decode batch of the serving benchmark (512 turns)
        dict(name="write-512", kind="write", T=512, hq=32, hkv=8),
        # one packed prefill at the engine's token budget
        dict(name="write-12288", kind="write", T=12288, hq=32, hkv=8),
        # one conversation alone on the card: latency, work split over its pages
        dict(name="decode-1x777", kind="decode", B=1, n=777, spread=0.0, hq=32, hkv=8),
        # the agents' batch: many short ragged conversations
        dict(name="decode-256x700", kind="decode", B=256, n=700, spread=0.9, hq=32, hkv=8),
        # few long contexts with 70B heads: the cache's stream is all there is
        dict(name="decode-8x32768", kind="decode", B=8, n=32768, spread=0.3, hq=64, hkv=8),
        # four small agents on one system prompt, smoke-size heads
        dict(name="shared-4x1024", kind="shared", B=4, groups=1, prefix=1024, tail=90, fp8=False, hq=8, hkv=2),
        # a team on one 2k system prompt, with short conversations behind it
        dict(name="shared-256x2048", kind="shared", B=256, groups=1, prefix=2048, tail=300, fp8=False, hq=32, hkv=8),
        # three agent kinds with 8k instructions each, quantised cache, largest batch
        dict(name="shared-512x8192-fp8", kind="shared", B=512, groups=3, prefix=8192, tail=300, fp8=True, hq=32, hkv=8),
        # one row's draw over the 8B vocabulary: latency
        dict(name="sample-1", kind="sample", B=1, V=128256, fp32=False, mix="all"),
        # the serving benchmark's batch, every filter in use
        dict(name="sample-512", kind="sample", B=512, V=128256, fp32=False, mix="all"),
        # 32-bit logits over the MoE model's vocabulary
        dict(name="sample-64-fp32", kind="sample", B=64, V=32000, fp32=True, mix="all"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "decode", "shared", "sample"])
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (8, 2), (2, 1), (8, 8), (8, 1)])
    if kind == "write":
        return dict(kind=kind, T=_log(rng, 1, 12288 * 48 // (hq + 2 * hkv) if hq > 32 else 12288), hq=hq, hkv=hkv)
    if kind == "decode":
        B = _log(rng, 1, 512)
        return dict(kind=kind, B=B, n=_log(rng, 1, min(32768, 262144 // B)), spread=round(rng.random(), 2), hq=hq, hkv=hkv)
    if kind == "shared":
        B = _log(rng, 2, 512)
        pages = _log(rng, 1, 128 if hq <= 32 else 64)
        return dict(kind=kind, B=B, groups=rng.randint(1, min(6, B)), prefix=PAGE * pages, tail=_log(rng, 1, 600 if B <= 256 else 300),
                    fp8=rng.random() < 0.5, hq=hq, hkv=hkv)
    fp32 = rng.random() < 0.4
    V = _log(rng, 100, 131072)
    return dict(kind=kind, B=_log(rng, 1, max(1, 512 * 128256 // V // (2 if fp32 else 1)) if V > 32000 else 512), V=V, fp32=fp32,
                mix=rng.choice(["all", "p", "k", "m", "t"]))


# ------------------------------------------------------------------ inputs

def _quant(x):
    """e4m3 codes and scale bytes of rows [..., HD] (see ``_plain_quant``)."""
    return _plain_quant(x.float())


def _cache(pages, hkv, fp8, gen):
    """A paged cache [pages, hkv, PAGE, HD] as a model fills it: keys with a few strong channels."""
    shape = (pages, hkv, PAGE, HD)
    k = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    strong = torch.ones(HD, device=DEV)
    strong[torch.randint(0, HD, (4,), generator=gen, device=DEV)] = 4.0
    k *= strong.to(k.dtype)
    v = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    if not fp8:
        return k, v, None, None
    parts = [[_quant(c) for c in t.split(max(1, 65536 // (hkv * PAGE)) * 4)] for t in (k, v)]
    (kc, ks), (vc, vs) = [[torch.cat([p[i] for p in ps]) for i in (0, 1)] for ps in parts]
    return kc.view(torch.float8_e4m3fn), vc.view(torch.float8_e4m3fn), ks, vs


def _queries(B, hq, hkv, gen):
    """Queries as the engine has them: a strided view of the packed projection."""
    packed = torch.empty(B, (hq + 2 * hkv) * HD, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    return packed[:, :hq * HD].view(B, hq, HD)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    kind, s = case["kind"], {"case": case}
    if kind == "write":
        T, hq, hkv = case["T"], case["hq"], case["hkv"]
        pages = (T + PAGE - 1) // PAGE + 3
        s["qkv"] = torch.empty(T, (hq + 2 * hkv) * HD, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
        s["qkv"] *= torch.exp(torch.empty((hq + 2 * hkv) * HD, device=DEV).normal_(generator=gen)).to(torch.bfloat16)
        s["slots"] = torch.randperm(pages * PAGE, generator=gen, device=DEV)[:T].to(torch.int32)
        s["positions"] = torch.randint(0, 8192, (T,), generator=gen, device=DEV).to(torch.int32)
        inv = 1.0 / (500000.0 ** (torch.arange(0, HD, 2, dtype=torch.float64, device=DEV) / HD))
        ang = torch.outer(torch.arange(8192, dtype=torch.float64, device=DEV), inv)
        s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=-1).float()
        for name in ("kcache", "vcache"):
            s[name] = torch.zeros(pages, hkv, PAGE, HD, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        for name in ("kscale", "vscale"):
            s[name] = torch.zeros(pages, hkv, PAGE, dtype=torch.uint8, device=DEV)
        return s
    if kind in ("decode", "shared"):
        B, hq, hkv = case["B"], case["hq"], case["hkv"]
        s["q"] = _queries(B, hq, hkv, gen)
        s["scale"] = 1.0 / math.sqrt(HD)
        if kind == "decode":
            least = max(1, int(case["n"] * (1.0 - case["spread"])))
            lens = torch.randint(least, case["n"] + 1, (B,), generator=gen, device=DEV)
            lens[0] = case["n"]
            group, prefix = torch.full((B,), -1, device=DEV), 0
        else:
            prefix = case["prefix"]
            # rows of one agent kind do not come in order; a row in twenty shares nothing
            group = torch.randint(0, case["groups"], (B,), generator=gen, device=DEV)
            group[torch.rand(B, generator=gen, device=DEV) < 0.05] = -1
            lens = torch.randint(1, case["tail"] + 1, (B,), generator=gen, device=DEV) + prefix * (group >= 0)
        most = prefix + case.get("tail", 0) if kind == "shared" else case["n"]
        width = (most + 8 + PAGE - 1) // PAGE
        shared = prefix // PAGE
        need = case.get("groups", 0) * shared + B * (width - shared)
        if kind == "shared":
            need += int((group < 0).sum()) * shared
        order = torch.randperm(need, generator=gen, device=DEV)
        table = torch.zeros(B, width, dtype=torch.int64, device=DEV)
        groups = case.get("groups", 0)
        heads, order = order[:groups * shared].view(groups, shared), order[groups * shared:]
        table[:, shared:], order = order[:B * (width - shared)].view(B, -1), order[B * (width - shared):]
        if shared:
            table[:, :shared] = heads[group.clamp_min(0)]
            table[group < 0, :shared] = order.view(-1, shared)
        s["kcache"], s["vcache"], s["kscale"], s["vscale"] = _cache(need, hkv, case.get("fp8", True), gen)
        s["page_table"], s["seq_lens"] = table.to(torch.int32), lens.to(torch.int32)
        if kind == "shared":
            s["group"] = group.to(torch.int32)
            s["group_lens"] = torch.full((case["groups"],), prefix, dtype=torch.int32, device=DEV)
        return s
    B, V = case["B"], case["V"]
    s["logits"] = torch.empty(B, V, dtype=torch.float32 if case["fp32"] else torch.bfloat16, device=DEV).normal_(generator=gen)
    s["logits"] *= 2.5                    # a head of likely tokens over a long tail
    s["uniform"] = torch.rand(B, generator=gen, device=DEV)

    def pick(values):
        return torch.tensor(values, device=DEV)[torch.randint(0, len(values), (B,), generator=gen, device=DEV)]

    mix = case["mix"]
    s["temperature"] = pick([0.6, 0.8, 1.0, 1.3] if mix != "all" else [0.0, 0.6, 0.8, 1.0, 1.3])
    s["top_k"] = (pick([0, 20, 50, 1000]) if mix in ("all", "k") else torch.zeros(B, device=DEV)).to(torch.int32)
    s["top_p"] = (pick([0.5, 0.9, 0.95, 1.0]) if mix in ("all", "p") else torch.ones(B, device=DEV)).float()
    s["min_p"] = (pick([0.0, 0.02, 0.05]) if mix in ("all", "m") else torch.zeros(B, device=DEV)).float()
    return s


# ------------------------------------------------------------- plain forms

def _times_pow2(x, e):
    """x * 2^e, exact: 2^e is put together from its bits, in two factors so that neither leaves the normal range."""
    half = torch.div(e, 2, rounding_mode="floor")
    for part in (half, e - half):
        x = x * ((part.int() + 127) << 23).view(torch.float32).unsqueeze(-1)
    return x


def _plain_quant(x):
    """Rows [..., HD] -> (e4m3 codes as bytes, scale bytes): the scale is 2^(byte - 127), the least power of two that brings
    the row's largest finite value to 448 or less; 0 in the exponent for a row of zeros."""
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(a)                                  # a = m * 2^e, 0.5 <= m < 1
    e = torch.where(m > 0.875, e - 8, e - 9)               # 448 = 0.875 * 2^9
    e = torch.where(a > 0, e, 0).clamp(-127, 127)
    y = _times_pow2(x, -e)
    y = torch.where(torch.isfinite(x), y, float("nan"))
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _plain_read(codes, scale):
    return _times_pow2(codes.view(torch.float8_e4m3fn).float(), scale.int() - 127)


def _plain_write(s):
    c, qkv = s["case"], s["qkv"]
    T, hq, hkv = c["T"], c["hq"], c["hkv"]
    rows = qkv.view(T, hq + 2 * hkv, HD).float()
    cs = s["cos_sin"][s["positions"].long()].unsqueeze(1)
    cos, sin = cs[..., :HD // 2], cs[..., HD // 2:]
    lo, hi = rows[:, :hq + hkv, :HD // 2], rows[:, :hq + hkv, HD // 2:]
    turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], dim=-1).to(torch.bfloat16)
    page, at = s["slots"].long() // PAGE, s["slots"].long() % PAGE
    back = []
    for cache, scale, x in ((s["kcache"], s["kscale"], turned[:, hq:].float()), (s["vcache"], s["vscale"], rows[:, hq + hkv:])):
        codes, e = _plain_quant(x)
        cache.view(torch.uint8)[page, :, at] = codes
        scale[page, :, at] = e
        back.append(_plain_read(cache.view(torch.uint8)[page, :, at], scale[page, :, at]).to(torch.bfloat16))
    return {"q": turned[:, :hq], "k": back[0], "v": back[1]}


def _plain_attention(s):
    c, q, table = s["case"], s["q"], s["page_table"].long()
    B, hq, hkv = c["B"], c["hq"], c["hkv"]

    def rows(cache, scale):               # [B, hkv, tokens, HD]
        x = cache.view(torch.uint8)[table] if scale is not None else cache[table]
        x = _plain_read(x, scale[table]) if scale is not None else x.float()
        return x.transpose(1, 2).reshape(B, hkv, -1, HD)

    k = rows(s["kcache"], s["kscale"])
    w = torch.matmul(q.float().reshape(B, hkv, hq // hkv, HD), k.transpose(-1, -2).contiguous()) * s["scale"]
    del k
    gone = torch.arange(w.shape[-1], device=DEV) >= s["seq_lens"].view(B, 1, 1, 1)
    w = w.masked_fill(gone, float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    return torch.matmul(w, rows(s["vcache"], s["vscale"])).reshape(B, hq, HD).to(q.dtype)


def _plain_sample(s):
    x = s["logits"].double() + 0.0        # -0 and +0 are one value
    B, V = x.shape
    x = torch.where(torch.isnan(x), float("-inf"), x)
    x, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    T = s["temperature"].double().unsqueeze(-1)
    w = torch.exp((x - x[:, :1]) / torch.where(T > 0, T, 1.0))
    w = torch.where(x == x[:, :1], 1.0, w)
    cum = w.cumsum(-1)
    k = s["top_k"].long().unsqueeze(-1)
    k = torch.where((k > 0) & (k < V), k, V)
    finite = (x > float("-inf")).sum(-1, keepdim=True).clamp_min(1)
    k = torch.minimum(k, finite)
    mass = cum.gather(-1, k - 1) * s["top_p"].double().unsqueeze(-1)
    n = torch.where(s["top_p"].unsqueeze(-1) < 1, ((cum - w) < mass).sum(-1, keepdim=True), V)
    n = torch.minimum(k, n)
    n = torch.minimum(n, (w >= s["min_p"].double().unsqueeze(-1)).sum(-1, keepdim=True)).clamp_min(1)
    n = torch.where(T > 0, n, 1)
    goal = s["uniform"].double().unsqueeze(-1) * cum.gather(-1, n - 1)
    r = torch.minimum((cum <= goal).sum(-1, keepdim=True), n - 1)
    return {"token": ids.gather(-1, r).squeeze(-1).to(torch.int32), "kept": n.squeeze(-1).to(torch.int32)}


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"write": _plain_write, "decode": _plain_attention, "shared": _plain_attention, "sample": _plain_sample}[kind](s)
    from calfkit_amd import ops

    if kind == "write":
        T, hq, hkv = c["T"], c["hq"], c["hkv"]
        q = torch.empty(T, hq, HD, dtype=torch.bfloat16, device=DEV)
        k, v = (torch.empty(T, hkv, HD, dtype=torch.bfloat16, device=DEV) for _ in range(2))
        ops.rope_qkv_write_fp8(s["qkv"], s["kcache"], s["vcache"], s["kscale"], s["vscale"], s["cos_sin"], s["positions"], s["slots"],
                               hq, hkv, q_out=q)
        ops.kv_read_fp8(k, v, s["kcache"], s["vcache"], s["kscale"], s["vscale"], s["slots"])
        return {"q": q, "k": k, "v": v}
    if kind == "sample":
        out, kept = (torch.empty(c["B"], dtype=torch.int32, device=DEV) for _ in range(2))
        ops.sample_filtered(out, s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["uniform"], kept=kept)
        return {"token": out, "kept": kept}
    out = torch.empty(c["B"], c["hq"], HD, dtype=torch.bfloat16, device=DEV)
    if kind == "decode":
        ops.attn_decode_fp8(out, s["q"], s["kcache"], s["vcache"], s["kscale"], s["vscale"], s["page_table"], s["seq_lens"], s["scale"])
    else:
        ops.attn_decode_shared(out, s["q"], s["kcache"], s["vcache"], s["page_table"], s["seq_lens"], s["group"], s["group_lens"],
                               s["scale"], kscale=s["kscale"], vscale=s["vscale"])
    return out


# ---------------------------------------------------------- least work, 64 bits

def work(case):
    kind = case["kind"]
    if kind == "write":
        T, hq, hkv = case["T"], case["hq"], case["hkv"]
        read = T * (hq + 2 * hkv) * HD * 2 + T * (HD * 4 + 8)
        cache = 2 * T * hkv * (HD + 1)
        return {"bytes": read + T * hq * HD * 2 + 2 * cache + 2 * T * hkv * HD * 2, "flops": 3 * T * (hq + 2 * hkv) * HD}
    if kind == "sample":
        return {"bytes": case["B"] * (case["V"] * (4 if case["fp32"] else 2) + 28), "flops": 4 * case["B"] * case["V"]}
    B, hq, hkv = case["B"], case["hq"], case["hkv"]
    token = hkv * 2 * (HD + 1 if case.get("fp8", True) else HD * 2)
    if kind == "decode":
        mean = case["n"] * (1.0 - case["spread"] / 2)
        read, seen = B * mean, B * mean
    else:
        tail = (case["tail"] + 1) / 2
        read = case["groups"] * case["prefix"] + B * tail
        seen = B * (0.95 * case["prefix"] + tail)
    return {"bytes": read * token + 2 * B * hq * HD * 2 + B * 8, "flops": 4 * seen * hq * HD}


def _two_to(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_quantised(x):
    """float64 rows -> the values that their e4m3 codes and scales stand for, from the format's definition."""
    a = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(a, -127)
    for lift in (128, 64, 32, 16, 8, 4, 2, 1):      # the largest exponent whose scale is still too small for the row, by halving
        e = torch.where(a > 448.0 * _two_to(e + lift - 1), e + lift, e)
    e = torch.where(a > 0, e, 0.0)
    y = x * _two_to(-e)
    octave = torch.frexp(y.abs().clamp_min(2.0 ** -6))[1] - 1
    return torch.round(y * _two_to(3 - octave)) * _two_to(octave - 3) * _two_to(e)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "sample":
        return None                        # whole numbers: equal or wrong
    if kind == "write":
        T, hq, hkv = case["T"], case["hq"], case["hkv"]
        x = s["qkv"].double().view(T, hq + 2 * hkv, 2, HD // 2)
        turn = torch.complex(*s["cos_sin"][s["positions"].long()].double().view(T, 1, 2, HD // 2).unbind(2))
        z = torch.complex(x[:, :hq + hkv, 0], x[:, :hq + hkv, 1]) * turn
        z = torch.cat([z.real, z.imag], dim=-1)
        # the cache holds the packed row's own bf16 values in fewer bits
        k = _exact_quantised(z[:, hq:].to(torch.bfloat16).double())
        return {"q": z[:, :hq], "k": k, "v": _exact_quantised(s["qkv"].double().view(T, -1, HD)[:, hq + hkv:])}
    B, hq, hkv = case["B"], case["hq"], case["hkv"]
    out = torch.zeros(B, hq, HD, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["seq_lens"].tolist()):
        pages = s["page_table"][b, :(n + PAGE - 1) // PAGE].long()
        kv = []
        for cache, scale in ((s["kcache"], s["kscale"]), (s["vcache"], s["vscale"])):
            x = (cache.view(torch.uint8) if scale is not None else cache)[pages]
            x = x.view(torch.float8_e4m3fn).double() * _two_to(scale[pages].int() - 127).unsqueeze(-1) if scale is not None else x.double()
            kv.append(x.permute(1, 0, 2, 3).reshape(hkv, -1, HD)[:, :n])
        p = torch.softmax(torch.matmul(s["q"][b].double().view(hkv, -1, HD), kv[0].transpose(1, 2).contiguous()) * s["scale"], dim=-1)
        out[b] = torch.matmul(p, kv[1]).view(hq, HD)
    return out
