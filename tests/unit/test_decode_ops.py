"""The quantised cache and the attention over it: kernels against 64-bit
formulas, on the GPU and (the reference implementations) on the CPU.

Tolerances are derived beside each check.  A rounding to bf16 is off by at
most 2^-8 of the value, one to e4m3 by 2^-4, one to fp32 by 2^-24.
"""

import math

import numpy as np
import pytest
import torch

from calfkit_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HD, PAGE = 128, 64


def _two_to(e: torch.Tensor) -> torch.Tensor:
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _quantised64(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The values an e4m3 row with a power-of-two scale holds, and the scale
    byte, from the format's definition in 64 bits (finite rows)."""
    x = x.double().cpu()
    a = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(a, -127)
    for lift in (128, 64, 32, 16, 8, 4, 2, 1):
        e = torch.where(a > 448.0 * _two_to(e + lift - 1), e + lift, e)
    e = torch.where(a > 0, e, 0.0)
    y = x * _two_to(-e)
    octave = torch.frexp(y.abs().clamp_min(2.0 ** -6))[1] - 1
    y = torch.round(y * _two_to(3 - octave)) * _two_to(octave - 3)
    return y * _two_to(e), (e.squeeze(-1) + 127).to(torch.uint8)


def _empty_cache(pages: int, hkv: int, device: str):
    def codes():
        return torch.zeros(pages, hkv, PAGE, HD, dtype=torch.uint8,
                           device=device).view(torch.float8_e4m3fn)

    def scales():
        return torch.full((pages, hkv, PAGE), 7, dtype=torch.uint8,
                          device=device)

    return codes(), codes(), scales(), scales()


def _values(cache: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """[P, hkv, PAGE, HD] in 64 bits, on the CPU."""
    return (cache.cpu().float().double()
            * _two_to(scale.cpu().int() - 127).unsqueeze(-1))


# ------------------------------------------------------------- e4m3 cache

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,hkv", [(1, 1), (1, 8), (7, 2), (65, 8), (300, 3)])
def test_kv_write_read_fp8(device, T, hkv):
    """Every stored value is the definition's, and reads back as it is."""
    g = torch.Generator().manual_seed(T * 31 + hkv)
    spread = torch.exp2(torch.randint(-30, 30, (T, hkv, 1), generator=g).float())
    rows = [(torch.randn(T, hkv, HD, generator=g) * spread).to(torch.bfloat16)
            for _ in range(2)]
    rows[0][0, 0] = 0.0                      # a row of zeros: scale 1
    rows[1][0, 0] = 0.0
    rows[1][0, 0, 5] = 448.0                 # the type's largest as it is
    rows[1][-1, -1] = torch.linspace(-1, 1, HD) * 2.0 ** -120
    if T > 2:
        rows[0][1, 0, :4] = torch.tensor([464.0, 1.0, -0.0, 2.0 ** -12])
        rows[0][2, 0] = 2.0 ** 119
    # a strided k, as a view of the packed rows
    packed = torch.zeros(T, 4 * hkv, HD, dtype=torch.bfloat16)
    packed[:, hkv:2 * hkv] = rows[0]
    k, v = packed.to(device)[:, hkv:2 * hkv], rows[1].to(device)
    pages = T // PAGE + 2
    kc, vc, ks, vs = _empty_cache(pages, hkv, device)
    slots = torch.randperm(pages * PAGE, generator=g)[:T].to(torch.int32)
    if T > 4:
        slots[3] = -1                        # padding
        slots[4] = pages * PAGE              # outside
    ops.kv_write_fp8(kc, vc, ks, vs, k, v, slots.to(device))
    keep = (slots >= 0) & (slots < pages * PAGE)
    s = slots[keep].long()
    for cache, scale, x in ((kc, ks, rows[0]), (vc, vs, rows[1])):
        want, byte = _quantised64(x[keep])
        assert torch.equal(scale.cpu()[s // PAGE, :, s % PAGE], byte)
        assert torch.equal(_values(cache, scale)[s // PAGE, :, s % PAGE], want)
        # what no slot names stays as it was
        other = torch.ones(pages * PAGE, dtype=torch.bool)
        other[s] = False
        o = torch.nonzero(other).squeeze(1)
        assert (scale.cpu()[o // PAGE, :, o % PAGE] == 7).all()
        assert (cache.view(torch.uint8).cpu()[o // PAGE, :, o % PAGE] == 0).all()
    back = [torch.full((T, hkv, HD), 3.0, dtype=torch.bfloat16, device=device)
            for _ in range(2)]
    ops.kv_read_fp8(*back, kc, vc, ks, vs, slots.to(device))
    for x, b in zip(rows, back):
        assert torch.equal(b.cpu().double()[keep], _quantised64(x[keep])[0])
        assert (b.cpu()[~keep] == 3.0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_kv_write_fp8_nonfinite(device):
    """NaN and infinities become NaN and leave their row's scale alone."""
    x = torch.randn(3, 1, HD).to(torch.bfloat16)
    y = x.clone()
    y[0, 0, 3], y[1, 0, 7], y[2, 0, 9] = math.nan, math.inf, -math.inf
    for at in ((0, 3), (1, 7), (2, 9)):
        x[at[0], 0, at[1]] = 0.0
    kc, vc, ks, vs = _empty_cache(1, 1, device)
    slots = torch.arange(3, dtype=torch.int32, device=device)
    ops.kv_write_fp8(kc, vc, ks, vs, x.to(device), y.to(device), slots)
    assert torch.equal(ks.cpu(), vs.cpu())
    k, v = _values(kc, ks)[0, 0, :3], _values(vc, vs)[0, 0, :3]
    bad = ~torch.isfinite(y[:, 0])
    assert torch.isnan(v[bad]).all() and torch.equal(v[~bad], k[~bad])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("q_out", [False, True])
@pytest.mark.parametrize("T,hq,hkv", [(1, 32, 8), (5, 2, 1), (130, 8, 2),
                                      (33, 12, 3)])
def test_rope_qkv_write_fp8(device, q_out, T, hq, hkv):
    g = torch.Generator().manual_seed(T)
    rows = torch.randn(T, (hq + 2 * hkv) * HD, generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 500, (T,), generator=g, dtype=torch.int32)
    table = ops.build_rope_table(500, HD)
    pages = T // PAGE + 1
    slots = torch.randperm(pages * PAGE, generator=g)[:T].to(torch.int32)
    if T > 1:
        slots[1] = -1
    kc, vc, ks, vs = _empty_cache(pages, hkv, device)
    qkv = rows.clone().to(device)
    q = torch.zeros(T, hq, HD, dtype=torch.bfloat16, device=device)
    ops.rope_qkv_write_fp8(qkv, kc, vc, ks, vs, table.to(device),
                           pos.to(device), slots.to(device), hq, hkv,
                           q_out=q if q_out else None)
    heads = rows.view(T, -1, HD).double()
    cos, sin = table[pos.long()].double().unsqueeze(1).split(HD // 2, -1)
    lo, hi = heads[:, :hq + hkv].split(HD // 2, -1)
    want = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    # two products and their sum in fp32 (3 roundings of values up to
    # |lo| + |hi|), one rounding to bf16
    mag = torch.cat([lo.abs() + hi.abs()] * 2, -1)
    tol = want.abs() * 2 ** -8 + mag * (3 * 2 ** -24)
    got = qkv.cpu().view(T, -1, HD)
    if q_out:
        assert torch.equal(qkv.cpu(), rows)
        turned_q = q.cpu()
    else:
        turned_q = got[:, :hq]
        assert ((got[:, :hq + hkv].double() - want).abs() <= tol).all()
        assert torch.equal(got[:, hq + hkv:], rows.view(T, -1, HD)[:, hq + hkv:])
    assert ((turned_q.double() - want[:, :hq]).abs() <= tol[:, :hq]).all()
    # the cache holds the packed row's own bf16 values, quantised
    again = rows.clone().to(device)
    ops.rope_qkv_write_fp8(again, *_empty_cache(pages, hkv, device),
                           table.to(device), pos.to(device), slots.to(device),
                           hq, hkv)
    packed = again.cpu().view(T, -1, HD)
    keep = slots >= 0
    s = slots[keep].long()
    for cache, scale, x in ((kc, ks, packed[:, hq:hq + hkv]),
                            (vc, vs, packed[:, hq + hkv:])):
        v, byte = _quantised64(x[keep])
        assert torch.equal(_values(cache, scale)[s // PAGE, :, s % PAGE], v)
        assert torch.equal(scale.cpu()[s // PAGE, :, s % PAGE], byte)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("splitk", [1, 4])
def test_rope_qkv_write_slab_fp8(device, splitk):
    T, Mp, hq, hkv = 19, 32, 8, 2
    W = (hq + 2 * hkv) * HD
    g = torch.Generator().manual_seed(splitk)
    work = torch.randn(splitk * Mp * W, generator=g)
    pos = torch.randint(0, 300, (T,), generator=g, dtype=torch.int32)
    table = ops.build_rope_table(300, HD)
    slots = torch.arange(T, dtype=torch.int32) * 3
    slots[4] = -1
    kc, vc, ks, vs = _empty_cache(1, hkv, device)
    qkv = torch.full((T, W), 9.0, dtype=torch.bfloat16, device=device)
    ops.rope_qkv_write_slab_fp8(qkv, work.to(device), kc, vc, ks, vs,
                                table.to(device), pos.to(device),
                                slots.to(device), hq, hkv, Mp, splitk)
    slabs = work.view(splitk, Mp, -1, HD)[:, :T].double()
    x, size = slabs.sum(0), slabs.abs().sum(0)
    cos, sin = table[pos.long()].double().unsqueeze(1).split(HD // 2, -1)
    lo, hi = x[:, :hq + hkv].split(HD // 2, -1)
    want = x.clone()
    want[:, :hq + hkv] = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    # splitk sums and 3 more roundings in fp32 of values up to size's pair,
    # one rounding to bf16
    pair = size[..., :64] + size[..., 64:]
    tol = want.abs() * 2 ** -8 + torch.cat([pair, pair], -1) * (splitk + 3) * 2 ** -24
    got = qkv.cpu().view(T, -1, HD)
    assert ((got.double() - want).abs() <= tol).all()
    keep = slots >= 0
    s = slots[keep].long()
    for cache, scale, part in ((kc, ks, got[:, hq:hq + hkv]),
                               (vc, vs, got[:, hq + hkv:])):
        assert torch.equal(_values(cache, scale)[0, :, s].transpose(0, 1),
                           _quantised64(part[keep])[0])


# -------------------------------------------------------------- attention

def _batch(lens, hq, hkv, *, seed=0, fp8=True, pages=None, width=None):
    """Caches, a shuffled page table and strided queries, on the CPU.  The
    table's unused entries name no page; the cache beyond a row is NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    need = [(n + PAGE - 1) // PAGE for n in lens]
    width = width or max(need + [1])
    pages = pages or sum(need) + 2
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((B, width), -1, dtype=torch.int32)
    k = torch.randn(pages, hkv, PAGE, HD, generator=g)
    v = torch.randn(pages, hkv, PAGE, HD, generator=g)
    used = torch.zeros(pages, PAGE, dtype=torch.bool)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            p = order.pop()
            table[b, i] = p
            used[p, :min(PAGE, n - i * PAGE)] = True
    k[~used.unsqueeze(1).expand(-1, hkv, -1)] = math.nan
    v[~used.unsqueeze(1).expand(-1, hkv, -1)] = math.nan
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    q = torch.randn(B, (hq + 2 * hkv) * HD, generator=g).to(torch.bfloat16)
    q = q[:, :hq * HD].view(B, hq, HD)
    s = dict(q=q, table=table, lens=torch.tensor(lens, dtype=torch.int32),
             k=k, v=v, ks=None, vs=None)
    if fp8:
        s["k"], s["v"], s["ks"], s["vs"] = _empty_cache(pages, hkv, "cpu")
        slots = torch.arange(pages * PAGE, dtype=torch.int32)
        ops.kv_write_fp8(s["k"], s["v"], s["ks"], s["vs"],
                         k.transpose(1, 2).reshape(-1, hkv, HD),
                         v.transpose(1, 2).reshape(-1, hkv, HD), slots)
    return s


def _to(s, device):
    out = {}
    for name, t in s.items():
        if t is None:
            out[name] = None
        elif name == "q":  # keep the packed rows' stride
            B, hq, _ = t.shape
            W = t.stride(0)
            base = torch.zeros(B, W, dtype=t.dtype)
            base[:, :hq * HD] = t.reshape(B, -1)
            out[name] = base.to(device)[:, :hq * HD].view(B, hq, HD)
        else:
            out[name] = t.to(device)
    return out


def _expect(s, scale):
    """out in 64 bits and how far a kernel may be from it.

    Scores: 128 products in fp32, each sum's rounding at most 2^-24 of the
    partial sums, so |ds| <= 2^-17 * scale * sum |q||k|, and the exponential
    and the joins' factors 2^-20 more; a weight is off by twice that.  Weights
    are rounded to bf16 (2^-8), sums of them and of their products in fp32.
    The output is rounded once.
    """
    B, hq, _ = s["q"].shape
    hkv = s["k"].shape[1]
    if s["ks"] is None:
        k, v = s["k"].double(), s["v"].double()
    else:
        k, v = _values(s["k"], s["ks"]), _values(s["v"], s["vs"])
    out = torch.zeros(B, hq, HD, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b, n in enumerate(s["lens"].tolist()):
        n = min(n, s["table"].shape[1] * PAGE)
        if n <= 0:
            continue
        pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
        kk, vv = (x[pages].permute(1, 0, 2, 3).reshape(hkv, -1, HD)[:, :n]
                  for x in (k, v))
        q = s["q"][b].double().view(hkv, -1, HD)
        p = torch.softmax(q @ kk.transpose(1, 2) * scale, -1)
        out[b] = (p @ vv).view(hq, HD)
        ds = 2 ** -17 * abs(scale) * (q.abs() @ kk.abs().transpose(1, 2)).amax()
        rel = 2 ** -8 + 2 * (ds + 2 ** -20) + n * 2 ** -24
        tol[b] = 2 ** -8 * out[b].abs() + rel * (p @ vv.abs()).view(hq, HD)
    return out, tol


def _close(got, want, tol):
    err = (got.cpu().double() - want).abs()
    assert not torch.isnan(err).any()
    assert (err <= tol).all(), float((err - tol).max())


def _decode(s, scale=HD ** -0.5, device="cpu"):
    d = _to(s, device)
    out = torch.full(s["q"].shape, 5.0, dtype=torch.bfloat16, device=device)
    ops.attn_decode_fp8(out, d["q"], d["k"], d["v"], d["ks"], d["vs"],
                        d["table"], d["lens"], scale)
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (32, 8), (64, 8), (16, 1),
                                    (9, 3)])
@pytest.mark.parametrize("lens", [[1], [64], [65], [0, 1, 63, 128, 200]])
def test_attn_decode_fp8(device, hq, hkv, lens):
    s = _batch(lens, hq, hkv, seed=hq)
    _close(_decode(s, device=device), *_expect(s, HD ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("B,n,hq,hkv", [(1, 5000, 32, 8), (3, 9001, 8, 8),
                                        (40, 700, 32, 8), (300, 130, 8, 2)])
def test_attn_decode_fp8_long_and_wide(B, n, hq, hkv):
    """Split sequences, ragged lengths, a table wider than any row."""
    rng = np.random.RandomState(B)
    lens = [int(x) for x in rng.randint(0, n + 1, B)]
    lens[0] = n
    s = _batch(lens, hq, hkv, seed=B, width=n // PAGE + 9)
    _close(_decode(s, device="cuda"), *_expect(s, HD ** -0.5))


@pytest.mark.parametrize("device", DEVICES)
def test_attn_decode_fp8_sharp_and_flat(device):
    """Scores of hundreds (one weight is all) and a scale of 0 (all equal)."""
    s = _batch([300, 77], 8, 2, seed=3)
    s["q"] = s["q"] * 40
    _close(_decode(s, 1.0, device=device), *_expect(s, 1.0))
    _close(_decode(s, 0.0, device=device), *_expect(s, 0.0))


@pytest.mark.parametrize("device", DEVICES)
def test_attention_with_a_negative_scale(device):
    """The smallest product weighs most, in the own tokens, in a prefix and
    where a row's end is masked."""
    s = _batch([300, 77, 1, 64], 8, 2, seed=6)
    _close(_decode(s, -0.3, device=device), *_expect(s, -0.3))
    for fp8 in (False, True):
        s = _shared_batch([0, 0, -1, 0], [128], [70, 1, 300, 33], 8, 2, seed=6,
                          fp8=fp8)
        s["glens"][0] = 100
        _close(_shared(s, device, -0.3), *_expect(s, -0.3))


@pytest.mark.parametrize("device", DEVICES)
def test_attn_decode_fp8_lengths_and_pages_out_of_range(device):
    """Lengths are taken to the table's width, negative ones are 0, and a page
    id outside the cache counts as a page without tokens."""
    s = _batch([128, 128, 100], 4, 2, seed=4)
    want, tol = _expect(s, HD ** -0.5)
    s["lens"] = torch.tensor([4000, 128, -3], dtype=torch.int32)
    want[2], tol[2] = 0.0, 0.0
    _close(_decode(s, device=device), want, tol)
    full = dict(s, lens=torch.tensor([64, 128, 0], dtype=torch.int32))
    want, tol = _expect(full, HD ** -0.5)
    s["table"][0, 1] = s["k"].shape[0]
    s["table"][1] = torch.tensor([-7, 1 << 30])
    want[1], tol[1] = 0.0, 0.0
    _close(_decode(s, device=device), want, tol)


@pytest.mark.parametrize("device", DEVICES)
def test_attn_decode_fp8_nan_row_stays_its_own(device):
    """A NaN key inside a row shows in that row and head alone."""
    s = _batch([70, 70], 4, 2, seed=5)
    want, tol = _expect(s, HD ** -0.5)
    page = int(s["table"][0, 1])
    s["k"].view(torch.uint8)[page, 1, 2, 9] = 0x7F
    got = _decode(s, device=device).cpu()
    assert torch.isnan(got[0, 2:]).all()
    got[0, 2:] = 0
    want[0, 2:], tol[0, 2:] = 0, 0
    _close(got, want, tol)


# --------------------------------------------------------- shared prefixes

def _shared_batch(groups, prefixes, tails, hq, hkv, *, seed=0, fp8=False):
    """Rows of group g share their first prefixes[g] tokens' pages."""
    B = len(groups)
    lens = [(prefixes[g] if g >= 0 else 0) + t for g, t in zip(groups, tails)]
    s = _batch(lens, hq, hkv, seed=seed, fp8=fp8)
    first = {}
    for b, g in enumerate(groups):
        if g < 0:
            continue
        lead = first.setdefault(g, b)
        # a row may be shorter than its prefix's last page: whole pages only
        n = prefixes[g] // PAGE
        s["table"][b, :n] = s["table"][lead, :n]
    s["group"] = torch.tensor(groups, dtype=torch.int32)
    s["glens"] = torch.tensor([p // PAGE * PAGE for p in prefixes],
                              dtype=torch.int32)
    return s


def _shared(s, device="cpu", scale=HD ** -0.5):
    d = _to(s, device)
    out = torch.full(s["q"].shape, 5.0, dtype=torch.bfloat16, device=device)
    ops.attn_decode_shared(out, d["q"], d["k"], d["v"], d["table"], d["lens"],
                           d["group"], d["glens"], scale, kscale=d["ks"],
                           vscale=d["vs"])
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hq,hkv", [(2, 1), (32, 8), (16, 1), (3, 3), (6, 2)])
def test_attn_decode_shared(device, fp8, hq, hkv):
    """Three interleaved groups, rows without one, tails of 0 and 1."""
    groups = [0, 1, -1, 0, 2, 0, 1, -1, 2]
    tails = [1, 70, 30, 0, 64, 63, 5, 0, 129]
    s = _shared_batch(groups, [64, 192, 320], tails, hq, hkv, seed=hq, fp8=fp8)
    _close(_shared(s, device), *_expect(s, HD ** -0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("B,ngroups,pages,hq,hkv", [
    (2, 1, 40, 32, 8), (100, 1, 9, 32, 8), (150, 64, 2, 8, 2),
    (70, 3, 17, 64, 8), (300, 5, 3, 2, 1)])
def test_attn_decode_shared_many(fp8, B, ngroups, pages, hq, hkv):
    """Tiles part full, split prefixes, as many groups as a call takes."""
    rng = np.random.RandomState(B)
    groups = [int(x) for x in rng.randint(-1, ngroups, B)]
    groups[0] = 0
    prefixes = [int(x) * PAGE for x in rng.randint(0, pages + 1, ngroups)]
    prefixes[0] = pages * PAGE
    tails = [int(x) for x in rng.randint(0, 150, B)]
    s = _shared_batch(groups, prefixes, tails, hq, hkv, seed=B, fp8=fp8)
    _close(_shared(s, "cuda"), *_expect(s, HD ** -0.5))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
def test_attn_decode_shared_any_prefix_length(device, fp8):
    """A prefix that ends inside a page, a row shorter than its prefix, a group
    id without a group, no groups at all: the result is the plain one."""
    s = _shared_batch([0, 0, 0, 1], [192, 64], [9, 40, 77, 3], 8, 2, fp8=fp8)
    s["lens"][1] = 150
    want = _expect(s, HD ** -0.5)
    for glens in ([100, 1], [192, 64], [0, 64], [191, -5], [1 << 30, 0]):
        if glens[0] > 192:     # a prefix past the rows' own: not common pages
            s["group"] = torch.tensor([0, -1, -1, -1], dtype=torch.int32)
        s["glens"] = torch.tensor(glens, dtype=torch.int32)
        _close(_shared(s, device), *want)
    s["group"] = torch.tensor([2, 77, -9, 1 << 30], dtype=torch.int32)
    _close(_shared(s, device), *want)
    s["glens"] = torch.zeros(0, dtype=torch.int32)
    _close(_shared(s, device), *want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("most", [2 ** 31 - 1, 2 ** 31 - 63, 2 ** 31 - 64])
def test_attn_decode_shared_longest_prefix_lengths(device, most):
    """The largest lengths an int32 holds: rows that end inside such a prefix
    are attended by themselves, the other groups as ever."""
    s = _shared_batch([0, 1, 0, 1, 1], [192, 128], [9, 40, 77, 3, 60], 8, 2)
    want = _expect(s, HD ** -0.5)
    for glens in ([most, 128], [192, most], [most, most]):
        s["glens"] = torch.tensor(glens, dtype=torch.int32)
        _close(_shared(s, device), *want)


@pytest.mark.parametrize("device", DEVICES)
def test_attn_decode_shared_short_rows_first(device):
    """A group's first rows may have ended: the entries past a row's length
    name other pages, and none of them is read."""
    s = _shared_batch([0, 0, 0, 0], [192], [9, 40, 77, 3], 8, 2)
    other = min(set(range(s["k"].shape[0])) - set(s["table"][2].tolist()))
    for b, n in ((0, 0), (1, 70), (3, 192)):
        s["lens"][b] = n
        s["table"][b, (n + PAGE - 1) // PAGE:] = other
    s["k"][other] = math.nan
    s["v"][other] = math.nan
    _close(_shared(s, device), *_expect(s, HD ** -0.5))


@pytest.mark.parametrize("device", DEVICES)
def test_attn_decode_shared_row_ends_inside_a_prefix_with_nan(device):
    """What lies in the common pages past a row's end does not reach it."""
    s = _shared_batch([0, 0, 0], [192], [9, 40, 77], 8, 2, fp8=False)
    s["lens"][0] = 100
    bad = int(s["table"][1, 1])              # tokens 64..127 of all rows
    s["v"][bad, :, 100 - PAGE + 1:] = math.inf
    s["k"][bad, :, 100 - PAGE + 1:] = math.nan
    got = _shared(s, device)
    assert not torch.isfinite(got[1:].float()).any()  # theirs to read
    s["v"][bad, :, 100 - PAGE + 1:] = 0
    s["k"][bad, :, 100 - PAGE + 1:] = 0
    want, tol = _expect(s, HD ** -0.5)
    _close(got[:1], want[:1], tol[:1])


@pytest.mark.gpu
@pytest.mark.parametrize("B", [4097, 65535])
def test_attn_decode_shared_most_rows(B):
    """Rows up to the limit, one group of them: every row is some tile's."""
    g = torch.Generator().manual_seed(B)
    s = _batch([2 * PAGE + 3], 1, 1, seed=3, fp8=False)
    s["q"] = torch.randn(B, 1, HD, generator=g).to(torch.bfloat16)
    s["table"] = s["table"].expand(B, -1).contiguous()
    s["lens"] = s["lens"].expand(B).contiguous()
    s["group"] = torch.arange(B, dtype=torch.int32) % 3 - 1
    s["glens"] = torch.tensor([128, 64], dtype=torch.int32)
    n = int(s["lens"][0])
    kk, vv = (s[x][s["table"][0].long()].double().view(-1, HD)[:n]
              for x in ("k", "v"))
    q = s["q"][:, 0].double()
    p = torch.softmax(q @ kk.T * HD ** -0.5, -1)
    want = p @ vv
    # as in _expect
    ds = 2 ** -17 * HD ** -0.5 * (q.abs() @ kk.abs().T).amax(-1, keepdim=True)
    rel = 2 ** -8 + 2 * (ds + 2 ** -20) + n * 2 ** -24
    tol = 2 ** -8 * want.abs() + rel * (p @ vv.abs())
    _close(_shared(s, "cuda")[:, 0], want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_cache_beyond_32_bit_offsets(fp8):
    """The last pages of a cache of more than 2^32 bytes (and elements of
    codes): written, read back, attended alone and with a shared prefix."""
    hkv = 8
    s = _shared_batch([0, 0, -1], [128], [30, 70, 100], 16, hkv, fp8=fp8)
    small = s["k"].shape[0]
    P = 66000 if fp8 else 33000
    assert P * hkv * PAGE * HD * s["k"].element_size() > 1 << 32
    d = _to(s, "cuda")
    for name in ("k", "v", "ks", "vs"):
        if d[name] is not None:
            t = torch.empty((P,) + s[name].shape[1:], dtype=s[name].dtype,
                            device="cuda")
            t[P - small:] = d[name]
            d[name] = t
    d["table"] += P - small
    want = _expect(s, HD ** -0.5)
    out = torch.full(s["q"].shape, 5.0, dtype=torch.bfloat16, device="cuda")
    ops.attn_decode_shared(out, d["q"], d["k"], d["v"], d["table"], d["lens"],
                           d["group"], d["glens"], HD ** -0.5, kscale=d["ks"],
                           vscale=d["vs"])
    _close(out, *want)
    if not fp8:
        return
    out.fill_(5.0)
    cache = (d["k"], d["v"], d["ks"], d["vs"])
    ops.attn_decode_fp8(out, d["q"], *cache, d["table"], d["lens"],
                        HD ** -0.5)
    _close(out, *want)
    g = torch.Generator().manual_seed(0)
    x = [torch.randn(5, hkv, HD, generator=g).to(torch.bfloat16)
         for _ in range(2)]
    slots = (P * PAGE - 1 - torch.arange(5)).to(torch.int32).cuda()
    ops.kv_write_fp8(*cache, x[0].cuda(), x[1].cuda(), slots)
    back = [torch.zeros_like(t, device="cuda") for t in x]
    ops.kv_read_fp8(*back, *cache, slots)
    for t, b in zip(x, back):
        assert torch.equal(b.cpu().double(), _quantised64(t)[0])


@pytest.mark.gpu
def test_attention_on_two_streams_at_once():
    """Calls in flight together have workspaces of their own."""
    batches = [_shared_batch([0, 0, 0, -1] * 4, [640], list(range(60, 76)), 32,
                             8, seed=i) for i in range(2)]
    moved = [_to(s, "cuda") for s in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    outs = [[torch.empty(s["q"].shape, dtype=torch.bfloat16, device="cuda")
             for _ in range(8)] for s in batches]
    torch.cuda.synchronize()
    for i in range(8):
        for d, stream, out in zip(moved, streams, outs):
            with torch.cuda.stream(stream):
                ops.attn_decode_shared(out[i], d["q"], d["k"], d["v"],
                                       d["table"], d["lens"], d["group"],
                                       d["glens"], HD ** -0.5,
                                       kscale=d["ks"], vscale=d["vs"])
    torch.cuda.synchronize()
    for s, out in zip(batches, outs):
        _close(out[0], *_expect(s, HD ** -0.5))
        for o in out[1:]:
            assert torch.equal(o, out[0])


def _integers(s, scale):
    """Small whole numbers for q and K, signs for V: scores are exact, so that
    what is left of _expect's bound is the weights'."""
    g = torch.Generator().manual_seed(7)
    q = s["q"]
    q.copy_(torch.randint(-1, 2, q.shape, generator=g).to(q.dtype))
    q[..., 40:] = 0
    for name, sc in (("k", "ks"), ("v", "vs")):
        x = torch.randint(0, 2, s[name].shape, generator=g) * 2 - 1
        if s[sc] is None:
            s[name].copy_(x.to(torch.bfloat16))
        else:
            s[name] = x.float().to(torch.float8_e4m3fn)
            s[sc].fill_(127)
    out, _ = _expect(s, scale)
    n = int(s["lens"].max())
    # a weight as two bf16 terms: 2^-7 of it is left to the second, whose own
    # rounding is 2^-8 of that.  Its exponent (up to 40 * scale * log2 e, below
    # 2^5) has two roundings of 2^-24, the exponential and a join's factor one
    # of 2^-23 each.  Twice, as the sum of weights is off by as much; sums of n
    # in fp32.  (sum of p |v| is 1)
    weight = 2 ** -15 + 2 ** -18 + 2 ** -22
    return out, 2 ** -8 * out.abs() + 2 * (weight + n * 2 ** -24)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hq,hkv", [(2, 1), (32, 8), (24, 3), (9, 1), (16, 1)])
def test_attention_weights_are_not_cut_to_bf16(device, hq, hkv):
    """Values of both signs that nearly cancel: a weight's error shows."""
    scale = 0.37
    s = _batch([260, 64, 1, 333], hq, hkv, seed=hq)
    want = _integers(s, scale)
    _close(_decode(s, scale, device=device), *want)
    for fp8 in (False, True):
        s = _shared_batch([0, 0, 1, -1, 0], [192, 320], [70, 1, 64, 300, 0],
                          hq, hkv, seed=hq, fp8=fp8)
        want = _integers(s, scale)
        _close(_shared(s, device, scale), *want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hq,hkv", [(8, 2), (16, 1)])
def test_attn_decode_shared_infinite_values_stay_infinite(device, hq, hkv):
    """An infinity in V is its row's output in that place, as the formula has
    it, in a prefix and among a row's own tokens."""
    s = _shared_batch([0, 0, -1], [128], [30, 70, 100], hq, hkv)
    want, tol = _expect(s, HD ** -0.5)
    first, own = int(s["table"][0, 1]), int(s["table"][2, 1])
    s["v"][first, 0, 5, 9] = math.inf
    s["v"][own, 0, 5, 77] = -math.inf
    got = _shared(s, device).cpu()
    heads = slice(0, hq // hkv)
    assert (got[:2, heads, 9] == math.inf).all()
    assert (got[2, heads, 77] == -math.inf).all()
    got[:2, heads, 9] = want[:2, heads, 9].to(got.dtype)
    got[2, heads, 77] = want[2, heads, 77].to(got.dtype)
    _close(got, want, tol)


def test_build_prefix_groups():
    table = np.array([[3, 4, 5, 6], [3, 4, 9, 0], [8, 1, 2, 0], [3, 4, 5, 7],
                      [8, 1, 2, 0], [11, 0, 0, 0], [3, 0, 0, 0]], np.int32)
    lens = np.array([250, 190, 192, 256, 130, 64, 63])
    group, glens = ops.build_prefix_groups(table, lens, max_groups=4)
    # rows 0, 1, 3 share pages 3, 4; rows 2, 4 share 8, 1 (row 4 has but two
    # whole pages); row 5 is alone and row 6 has no whole page
    a, b = group[0], group[2]
    assert a >= 0 and b >= 0 and a != b
    assert group.tolist() == [a, a, b, a, b, -1, -1]
    assert glens[a] == 128 and glens[b] == 128
    one, lens1 = ops.build_prefix_groups(table, lens, max_groups=1)
    assert one.tolist() == [0, 0, -1, 0, -1, -1, -1] and lens1.tolist() == [128]
    none, _ = ops.build_prefix_groups(table, lens, min_rows=4)
    assert (none == -1).all()
    # (3 - 1) * 2 + (2 - 1) * 2 page reads are saved
    for least, some in ((6, True), (7, False)):
        group, _ = ops.build_prefix_groups(table, lens, min_saved=least)
        assert bool((group >= 0).any()) == some
    none, _ = ops.build_prefix_groups(table[:0], lens[:0])
    assert none.shape == (0,)


def _agent_rows(kinds, per, common, own, tail):
    """Rows of several kinds: `common` pages for all, `own` pages of each
    kind, `tail` of each row; in shuffled order."""
    ids = iter(range(1 << 20))

    def take(n):
        return [next(ids) for _ in range(n)]

    head, rows = take(common), []
    for _ in range(kinds):
        kind = head + take(own)
        rows += [kind + take(tail) for _ in range(per)]
    rows = np.array(rows, np.int32)
    return rows[np.random.RandomState(kinds).permutation(len(rows))]


def _pages_saved(table, lens, group, glens):
    """After checking that every group is one."""
    saved = 0
    assert group.max(initial=-1) < len(glens)
    for g, n in enumerate(glens):
        rows = np.flatnonzero(group == g)
        if rows.size == 0:
            assert n == 0
            continue
        assert rows.size >= 2 and n > 0 and n % 64 == 0
        assert (lens[rows] >= n).all()
        assert (table[rows, :n // 64] == table[rows[0], :n // 64]).all()
        saved += (rows.size - 1) * (n // 64)
    return saved


def test_prefix_groups_past_a_common_first_page():
    """Three kinds with 8192 instructions each behind one page of preamble:
    three groups, not one of the preamble."""
    table = _agent_rows(3, 32, 1, 127, 3)
    lens = np.full(96, 131 * 64 - 10)
    group, glens = ops.build_prefix_groups(table, lens, max_groups=16)
    assert sorted(glens[glens > 0]) == [8192] * 3
    assert np.bincount(group).tolist() == [32] * 3
    assert _pages_saved(table, lens, group, glens) == 3 * 31 * 128


def test_prefix_groups_leave_a_short_row_out():
    """One row that ends early does not cut the others' prefix."""
    table = _agent_rows(1, 96, 0, 128, 1)
    lens = np.full(96, 128 * 64 + 30)
    for short in (70, 20):                 # one whole page, none
        lens[17] = short
        group, glens = ops.build_prefix_groups(table, lens, max_groups=16,
                                               min_saved=94 * 128)
        assert glens[glens > 0].tolist() == [8192]
        assert np.flatnonzero(group < 0).tolist() == [17]
    # two such rows are a group of their own
    lens[17] = lens[40] = 70
    group, glens = ops.build_prefix_groups(table, lens, max_groups=16)
    assert glens[:3].tolist() == [8192, 64, 0]
    assert np.flatnonzero(group == 1).tolist() == [17, 40]
    group, glens = ops.build_prefix_groups(table, lens, min_rows=3)
    assert np.flatnonzero(group < 0).tolist() == [17, 40]
    group, glens = ops.build_prefix_groups(table, lens, min_pages=2)
    assert np.flatnonzero(group < 0).tolist() == [17, 40]


def test_prefix_groups_of_unrelated_rows_and_of_too_many_kinds():
    rows = _agent_rows(40, 1, 0, 5, 1)
    group, glens = ops.build_prefix_groups(rows, np.full(40, 380))
    assert (group == -1).all() and (glens == 0).all()
    table = _agent_rows(6, 4, 0, 9, 1)
    lens = np.full(24, 9 * 64 + 5)
    group, glens = ops.build_prefix_groups(table, lens, max_groups=4)
    assert glens.tolist() == [9 * 64] * 4
    assert np.bincount(group + 1).tolist() == [8, 4, 4, 4, 4]
    none, glens = ops.build_prefix_groups(table, lens, max_groups=0)
    assert (none == -1).all() and glens.size == 0


def _most_saved(table, whole, rows, depth, given):
    """The most page reads that groups of these rows can save, each row left
    over worth `given` (its place in a group around): by trying both."""
    if len(rows) == 1:
        return given
    while all(whole[r] > depth for r in rows) and len(
            {table[r, depth] for r in rows}) == 1:
        depth += 1
    kinds = {}
    for r in rows:
        if whole[r] > depth:
            kinds.setdefault(table[r, depth], []).append(r)
    here = len(rows) - sum(map(len, kinds.values()))

    def total(each):
        return here * each + sum(_most_saved(table, whole, k, depth, each)
                                 for k in kinds.values())

    return max(total(given), total(depth) - depth if depth else 0)


def test_prefix_groups_save_nearly_the_most():
    """Random trees of runs: every group is one, and all together save what the
    best one of them does or more (it is taken first, and each further one
    adds), on average 99 % of what any choice can."""
    rng = np.random.RandomState(0)
    shares = []
    for _ in range(400):
        B, W, kinds = rng.randint(1, 14), rng.randint(1, 9), rng.randint(1, 4)
        ids, table = {}, np.zeros((B, W), np.int32)
        for b in range(B):
            path = ()
            for j in range(W):
                path += (rng.randint(kinds) if rng.rand() < 0.5 else 0,)
                table[b, j] = ids.setdefault(path, len(ids))
        lens = rng.randint(0, W * 64 + 130, B)
        saved = _pages_saved(table, lens, *ops.build_prefix_groups(table, lens))
        whole = np.minimum(lens // 64, W)
        runs = {}
        for b in range(B):
            for n in range(1, whole[b] + 1):
                runs.setdefault(tuple(table[b, :n]), []).append(n)
        one = max([(len(r) - 1) * r[0] for r in runs.values()], default=0)
        most = _most_saved(table, whole, list(range(B)), 0, 0)
        assert one <= saved <= most
        if most:
            shares.append(saved / most)
    assert np.mean(shares) >= 0.99


# --------------------------------------------------------------- refusals

def _refusal_args(device):
    s = _to(_batch([70, 5], 4, 2, seed=1), device)
    qkv = torch.zeros(2, 8 * HD, dtype=torch.bfloat16, device=device)
    i32 = torch.zeros(2, dtype=torch.int32, device=device)
    rows = torch.zeros(2, 2, HD, dtype=torch.bfloat16, device=device)
    table = ops.build_rope_table(8, HD, device=device)
    cache = (s["k"], s["v"], s["ks"], s["vs"])
    out = torch.zeros(2, 4, HD, dtype=torch.bfloat16, device=device)
    return s, cache, qkv, i32, rows, table, out


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    s, cache, qkv, i32, rows, table, out = _refusal_args(device)
    kc, vc, ks, vs = cache

    def refused(call, *args, **kw):
        with pytest.raises(RuntimeError):
            call(*args, **kw)

    bf16 = torch.zeros(kc.shape, dtype=torch.bfloat16, device=device)
    w, r = ops.kv_write_fp8, ops.kv_read_fp8
    refused(w, bf16, vc, ks, vs, rows, rows, i32)
    refused(w, kc[:, :1], vc, ks, vs, rows, rows, i32)
    refused(w, kc, vc, ks[:1], vs, rows, rows, i32)
    refused(w, kc, vc, ks.int(), vs, rows, rows, i32)
    refused(w, kc, vc, ks, vs, rows.float(), rows, i32)
    refused(w, kc, vc, ks, vs, rows[:, :1], rows, i32)
    refused(w, kc, vc, ks, vs, rows, rows, i32.long())
    refused(w, kc, vc, ks, vs, rows, rows, i32[:1])
    refused(w, kc, vc, ks, vs, rows.transpose(1, 2).contiguous()
            .transpose(1, 2), rows, i32)
    refused(r, rows, rows, kc, vc, ks, vs, i32[:1])
    refused(r, rows, rows[..., :64], kc, vc, ks, vs, i32)
    rope = ops.rope_qkv_write_fp8
    refused(rope, qkv, kc, vc, ks, vs, table, i32, i32, 5, 2)
    refused(rope, qkv, kc, vc, ks, vs, table, i32, i32, 6, 1)
    refused(rope, qkv.float(), kc, vc, ks, vs, table, i32, i32, 4, 2)
    refused(rope, qkv, kc, vc, ks, vs, table[:, :64], i32, i32, 4, 2)
    refused(rope, qkv, kc, vc, ks, vs, table, i32.long(), i32, 4, 2)
    refused(rope, qkv, kc, vc, ks, vs, table, i32, i32, 4, 2, q_out=out.float())
    if device == "cuda":  # 16 B accesses
        odd = torch.zeros(qkv.numel() + 1, dtype=qkv.dtype, device=device)
        refused(rope, odd[1:].view(qkv.shape), kc, vc, ks, vs, table, i32, i32,
                4, 2)
        shifted = torch.zeros(kc.numel() + 1, dtype=torch.uint8, device=device)
        shifted = shifted[1:].view(torch.float8_e4m3fn).view(kc.shape)
        refused(w, shifted, vc, ks, vs, rows, rows, i32)
    refused(ops.rope_qkv_write_slab_fp8, qkv,
            torch.zeros(8 * HD * 2, device=device), kc, vc, ks, vs, table,
            i32, i32, 4, 2, 2, 2)
    dec = ops.attn_decode_fp8
    q, t, n = s["q"], s["table"], s["lens"]
    refused(dec, out, q.float(), kc, vc, ks, vs, t, n, 1.0)
    refused(dec, out[:1], q, kc, vc, ks, vs, t, n, 1.0)
    refused(dec, out, q, bf16, bf16, ks, vs, t, n, 1.0)
    refused(dec, out, q, kc, vc, ks, vs, t.long(), n, 1.0)
    refused(dec, out, q, kc, vc, ks, vs, t[:1], n, 1.0)
    refused(dec, out, q, kc, vc, ks, vs, t, n.long(), 1.0)
    refused(dec, out[:, :3].contiguous(), q[:, :3], kc, vc, ks, vs, t, n, 1.0)
    refused(dec, out, q, kc[:0], vc[:0], ks[:0], vs[:0], t, n, 1.0)
    none = out[:, :0].contiguous()
    refused(dec, none, none, kc, vc, ks, vs, t, n, 1.0)
    wide = torch.zeros(2, 34, HD, dtype=torch.bfloat16, device=device)
    refused(dec, wide, wide, kc, vc, ks, vs, t, n, 1.0)
    sh = ops.attn_decode_shared
    g, gl = i32, i32[:1]
    refused(sh, out, q, kc, vc, t, n, g, gl, 1.0)            # e4m3, no scales
    refused(sh, out, q, bf16, bf16, t, n, g, gl, 1.0, kscale=ks)
    refused(sh, out, q, bf16, bf16, t, n, g, gl, 1.0, kscale=ks, vscale=vs)
    refused(sh, out, q, bf16, bf16, t, n, g[:1], gl, 1.0)
    refused(sh, out, q, bf16[:0], bf16[:0], t, n, g, gl, 1.0)
    refused(sh, out, q, bf16, bf16, t, n, g, gl.long(), 1.0)
    refused(sh, out, q, bf16, bf16, t, n, g,
            torch.zeros(65, dtype=torch.int32, device=device), 1.0)


@pytest.mark.parametrize("device", DEVICES)
def test_empty_batches(device):
    s, cache, qkv, i32, rows, table, out = _refusal_args(device)
    kc, vc, ks, vs = cache
    before = kc.view(torch.uint8).clone()
    ops.kv_write_fp8(kc, vc, ks, vs, rows[:0], rows[:0], i32[:0])
    ops.kv_read_fp8(rows[:0], rows[:0], kc, vc, ks, vs, i32[:0])
    ops.rope_qkv_write_fp8(qkv[:0], kc, vc, ks, vs, table, i32[:0], i32[:0],
                           4, 2)
    assert torch.equal(kc.view(torch.uint8), before)
    ops.attn_decode_fp8(out[:0], s["q"][:0], kc, vc, ks, vs, s["table"][:0],
                        s["lens"][:0], 1.0)
    ops.attn_decode_shared(out[:0], s["q"][:0], kc, vc, s["table"][:0],
                           s["lens"][:0], i32[:0], i32[:1], 1.0, kscale=ks,
                           vscale=vs)
