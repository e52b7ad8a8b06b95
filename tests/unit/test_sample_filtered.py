"""Filtered draws from given random numbers: every token and kept count is the
formula's in 64 bits, compared for equality.  A row whose random number or
top-p lies nearer a border than 64-bit sums of its length can tell is left out
(``_check`` derives the distance).
"""

import math

import pytest
import torch

from calfkit_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _formula(x, T, k, p, mp, u):
    """(token, kept, how near the nearest border is, relative to the sum) by
    explicit ranks in 64 bits; python floats, no torch sums."""
    V = x.numel()
    x = [float(v) for v in x]
    order = sorted((i for i in range(V) if x[i] > -math.inf),
                   key=lambda i: (-x[i], i))
    if not order:
        return 0, 1, 1.0
    if not T > 0:
        return order[0], 1, 1.0
    m = x[order[0]]
    w = [1.0 if x[i] == m else math.exp((x[i] - m) / T) for i in order]
    n = min(k if 0 < k < V else V, len(order))
    near = 1.0
    if p < 1:
        total = math.fsum(w[:n])
        goal, before, np_ = p * total, 0.0, 0
        sums = []
        for wi in w:
            sums.append(before)
            before += wi
        np_ = sum(s < goal for s in sums)
        # an exact tie of whole sums (equal weights of 1) is no near miss
        near = min([near] + [abs(s - goal) / total for s in sums
                             if s != goal or s != int(s)])
        n = min(n, np_)
    n = max(1, min(n, sum(wi >= mp for wi in w)))
    total = math.fsum(w[:n])
    goal, cum, r = min(u, 1 - 2.0 ** -53) * total, 0.0, 0
    for r in range(n):
        cum += w[r]
        if cum != goal or cum != int(cum):
            near = min(near, abs(cum - goal) / total)
        if cum > goal:
            break
    return order[r], n, near


def _check(logits, T, k, p, mp, u, device):
    B, V = logits.shape
    dev = [torch.tensor(t, dtype=d, device=device)
           for t, d in ((T, torch.float32), (k, torch.int32),
                        (p, torch.float32), (mp, torch.float32),
                        (u, torch.float32))]
    x = logits.to(device)
    before = x.clone()
    out = torch.full((B,), -5, dtype=torch.int32, device=device)
    kept = torch.full((B,), -5, dtype=torch.int32, device=device)
    ops.sample_filtered(out, x, *dev, kept=kept)
    same = torch.equal(x.view(torch.uint8), before.view(torch.uint8))
    assert same, "logits are not to be changed"
    only = torch.full((B,), -5, dtype=torch.int32, device=device)
    ops.sample_filtered(only, x, *dev)
    assert torch.equal(only, out)
    f32 = [t.cpu() for t in dev]
    for b in range(B):
        if u[b] < 0:
            assert int(out[b]) == int(kept[b]) == -5
            continue
        token, n, near = _formula(logits[b], float(f32[0][b]), int(f32[1][b]),
                                  float(f32[2][b]), float(f32[3][b]),
                                  float(f32[4][b]))
        # V additions of relative 2^-53, weights of relative 2^-50 and of
        # absolute 2^-44 (fixed point) each: below V * 2^-43 of a sum >= 1
        if near <= V * 2.0 ** -43:
            continue
        got = (int(out[b]), int(kept[b]))
        assert got == (token, n), (b, T[b], k[b], p[b], mp[b], u[b])


def _filters(rng, B):
    def pick(values):
        return [values[int(torch.randint(0, len(values), (1,), generator=rng))]
                for _ in range(B)]

    return (pick([0.0, 0.3, 0.7, 1.0, 1.5, 20.0]),
            pick([0, -1, 1, 5, 40, 1000]),
            pick([0.0, 0.3, 0.9, 0.999, 1.0, 1.5]),
            pick([0.0, 0.01, 0.1, 1.0, 2.0]),
            torch.rand(B, generator=rng).tolist())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1, 2, 7, 64, 999, 4096])
def test_filters(device, dtype, V):
    rng = torch.Generator().manual_seed(V)
    B = 24
    x = (torch.randn(B, V, generator=rng) * 3).to(dtype)
    T, k, p, mp, u = _filters(rng, B)
    u[0], u[1], u[2] = 0.0, 1 - 2.0 ** -24, -1.0
    _check(x, T, k, p, mp, u, device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,V,B", [
    (torch.bfloat16, 128256, 12), (torch.bfloat16, 32000, 12),
    (torch.bfloat16, 32761, 6), (torch.bfloat16, 140001, 4),
    (torch.float32, 32000, 12), (torch.float32, 128256, 4),
    (torch.float32, 70003, 4)])
def test_vocabularies(dtype, V, B):
    """Real vocabularies, odd sizes (rows that start off 16 bytes), rows
    longer than the registers hold; half the rows unfiltered."""
    rng = torch.Generator().manual_seed(V + B)
    x = (torch.randn(B, V, generator=rng) * 2.5).to(dtype)
    T, k, p, mp, u = _filters(rng, B)
    for b in range(0, B, 2):
        k[b], p[b], mp[b] = 0, 1.0, 0.0
        T[b] = [0.7, 1.0, 1.5][b % 3]
    _check(x, T, k, p, mp, u, "cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows(device, dtype):
    """Masks of -inf, of the type's lowest and of other large negative values,
    NaN entries, rows that are all masked, infinities, zeros of both signs."""
    rng = torch.Generator().manual_seed(3)
    V = 500
    x = (torch.randn(16, V, generator=rng) * 2).to(dtype)
    low = torch.finfo(dtype).min
    off = torch.rand(V, generator=rng) < 0.8
    for b, v in enumerate((-math.inf, low, -1e4, -1e9, -65536.0, math.nan)):
        x[b, off] = v
    x[6] = -math.inf
    x[7] = math.nan
    x[8] = low
    x[9, 10], x[9, 300] = math.inf, math.inf
    x[10] = 0.0
    x[10, ::2] = -0.0
    x[11] = -math.inf
    x[11, 77] = -3.0
    x[12] = 1.0                     # one value: ranks are the indices
    x[13, :250] = -1e9
    x[14] *= 1e30
    x[15] *= 1e-30
    for T, k, p, mp in ((1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0),
                        (1.0, 450, 1.0, 0.0), (1.3, 0, 0.5, 0.02),
                        (1e4, 300, 0.999, 0.0), (1e-3, 0, 0.95, 0.0)):
        u = torch.rand(16, generator=rng).tolist()
        _check(x, [T] * 16, [k] * 16, [p] * 16, [mp] * 16, u, device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ties(device, dtype):
    """Few distinct values: borders inside runs of equal logits."""
    rng = torch.Generator().manual_seed(9)
    V, B = 3001, 20
    x = torch.randint(-3, 4, (B, V), generator=rng).to(dtype)
    T, k, p, mp, u = _filters(rng, B)
    k = [0, 1, 2, 300, 500, 3000, 700, 100, 0, 429] * 2
    T = [t if t > 0 else 1.0 for t in T]
    _check(x, T, k, p, mp, u, device)


@pytest.mark.gpu
def test_general_search_rows():
    """Rows that fit neither histogram: more distinct bf16 values than its
    list holds, tiny values beside large ones, thousands of members in one
    bin."""
    bits = torch.arange(0, 1 << 15, 3, dtype=torch.int32).to(torch.int16)
    many = bits.view(torch.bfloat16)
    many = many[torch.isfinite(many)].clone()
    many = torch.cat([many[many < 80.0], -many[many < 1e6]])
    V = many.numel()
    rng = torch.Generator().manual_seed(1)
    x = torch.stack([many, many[torch.randperm(V, generator=rng)],
                     (torch.randn(V, generator=rng)).to(torch.bfloat16)])
    x[2, 5], x[2, 6] = 1e-30, -1e-30
    f = [1.0, 0.8, 1.0], [0, 100, 0], [0.95, 1.0, 0.9], [0.0, 0.0, 0.01]
    _check(x, *f, [0.31, 0.77, 0.52], "cuda")
    y = torch.zeros(3, 5000)
    y[1, 100:] = -7.0
    y[2, :2500] = torch.randn(2500, generator=rng) * 1e-6
    y[2, 2500:] = -10.0
    _check(y, [1.0, 1.0, 0.9], [0, 3000, 0], [0.5, 0.9, 1.0], [0.0] * 3,
           [0.4, 0.999, 0.2], "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("p", [0.0, -1.0])
def test_general_search_of_rows_that_keep_one(p):
    """top_p of 0 and less, over rows that no histogram holds."""
    rng = torch.Generator().manual_seed(2)
    x = (torch.randn(6, 5000, generator=rng)).to(torch.bfloat16)
    x[:, 5] = 1e-30
    x[3:] = x[3:, :1]                       # equal but for that one
    x[3:, 5] = 1e-30
    y = torch.zeros(6, 5000)
    y[1:, 100:] = -7.0
    y[3:, :2500] = torch.randn(2500, generator=rng) * 1e-6
    y[3:, 2500:] = -10.0
    for rows in (x, y):
        _check(rows, [1.0, 0.9, 30.0] * 2, [0, 3, 4000] * 2, [p] * 6,
               [0.0, 0.0, 0.5] * 2, [0.0, 0.6, 1 - 2.0 ** -24] * 2, "cuda")


# one logit of 0 over 2000 of -c: with u these draw near a border, 2^-39 to
# 2^-35 of the sum away from it.  A fixed point of 2^-43, whatever the row's
# length, moves the sum of 2000 by up to 2^-33 and draws another token.
NEAR_BORDERS = [(13.122835159301758, 0.9983434081077576),
                (14.66104507446289, 0.9997100234031677),
                (14.730710983276367, 0.9996070861816406),
                (14.563593864440918, 0.9998524785041809),
                (14.459906578063965, 0.9994561672210693),
                (13.302825927734375, 0.9992644190788269)]


@pytest.mark.parametrize("device", DEVICES)
def test_fp32_draws_near_a_border(device):
    V = 2001
    x = torch.zeros(len(NEAR_BORDERS), V)
    x[:, 1:] = -torch.tensor([c for c, _ in NEAR_BORDERS])[:, None]
    u = [u for _, u in NEAR_BORDERS]
    one = torch.ones(len(u), device=device)
    none = torch.zeros(len(u), dtype=torch.int32, device=device)
    out = none.clone()
    ops.sample_filtered(out, x.to(device), one, none, one, 0 * one,
                        torch.tensor(u, device=device))
    for b, u in enumerate(u):
        token, _, near = _formula(x[b], 1.0, 0, 1.0, 0.0, u)
        # 2000 weights of 2^-18 and less and their sums in steps of 2^-51, each
        # off by half of one, and a 64-bit sum to the border: 2^-40
        assert 2.0 ** -39 < near < 2.0 ** -35
        assert int(out[b]) == token


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets():
    """The last rows of logits of more than 2^32 bytes; the others, not drawn,
    keep their outputs."""
    B, V = 17000, 128256
    assert B * V * 2 > 1 << 32
    g = torch.Generator().manual_seed(1)
    last = (torch.randn(2, V, generator=g) * 3).to(torch.bfloat16)
    logits = torch.empty(B, V, dtype=torch.bfloat16, device="cuda")
    logits[-2:] = last.cuda()
    f = [torch.full((B,), v, dtype=d, device="cuda")
         for v, d in ((0.8, torch.float32), (500, torch.int32),
                      (0.9, torch.float32), (0.001, torch.float32),
                      (-1.0, torch.float32))]
    f[4][-2:] = torch.tensor([0.3, 0.8])
    out, kept = (torch.full((B,), -7, dtype=torch.int32, device="cuda")
                 for _ in range(2))
    ops.sample_filtered(out, logits, *f, kept=kept)
    want, n = (torch.zeros(2, dtype=torch.int32) for _ in range(2))
    ops.sample_filtered(want, last, *[t[-2:].cpu() for t in f], kept=n)
    assert torch.equal(out[-2:].cpu(), want)
    assert torch.equal(kept[-2:].cpu(), n)
    assert (out[:-2] == -7).all() and (kept[:-2] == -7).all()


@pytest.mark.gpu
def test_view_off_alignment():
    """Logits that start off 16 bytes."""
    for dtype in (torch.bfloat16, torch.float32):
        base = (torch.randn(5 * 777 + 3) * 2).to(dtype)
        x = base[3:].view(5, 777)
        dev = base.cuda()[3:].view(5, 777)
        assert dev.data_ptr() % 16 != 0
        out = torch.empty(5, dtype=torch.int32, device="cuda")
        u = torch.tensor([0.1, 0.3, 0.5, 0.7, 0.9])
        one = torch.ones(5, device="cuda")
        zero = torch.zeros(5, dtype=torch.int32, device="cuda")
        ops.sample_filtered(out, dev, one, zero, one, 0 * one,
                            u.cuda())
        want = [_formula(x[b], 1.0, 0, 1.0, 0.0, float(u[b]))[0]
                for b in range(5)]
        assert out.tolist() == want


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    V, B = 50, 3
    x = torch.zeros(B, V, device=device)
    f = torch.ones(B, device=device)
    i = torch.zeros(B, dtype=torch.int32, device=device)

    def refused(*args, **kw):
        with pytest.raises(RuntimeError):
            ops.sample_filtered(*args, **kw)

    refused(i, x.half(), f, i, f, f, f)
    refused(i, x.t().contiguous().t(), f, i, f, f, f)
    refused(i, x[0], f, i, f, f, f)
    refused(i.long(), x, f, i, f, f, f)
    refused(i, x, f.double(), i, f, f, f)
    refused(i, x, f, i.long(), f, f, f)
    refused(i, x, f, i, f[:2], f, f)
    refused(i, x, f, i, f, f, f, kept=i.long())
    refused(i, x[:, :0], f, i, f, f, f)
    ops.sample_filtered(i[:0], x[:0], f[:0], i[:0], f[:0], f[:0], f[:0])
