"""The 8-bit key/value cache on the GPU against its definition: codes and scales bit for bit in numpy's fp32, attention
and probabilities against 64 bits.

Tolerances of the attention, derived from its arithmetic:
  fp16 outputs      half a step: |x| 2^-11, and 2^-25 where x is subnormal
  scores            64 products of exact operands summed in fp32, each partial sum off by at most 2^-23 of sum |q k|
                    (a truncated step), then two fp32 products: |ds| <= 2^-16 A, A the largest scale ks sum |q k8|; the
                    exponent's argument s log2(e) is rounded once more, |s| <= A
  probabilities     relative 2 |ds| (numerator and sum), 2^-20 for two exponentials and the division, and
                    (n / 4 + 64) 2^-23 for the sum of n terms
  out               the probabilities' error times the largest |v|, and as much again for the sum of products
"""
import numpy as np
import pytest
import torch

import mimizuku_b200 as m

pytestmark = pytest.mark.gpu

HD = 64
KINDS = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def cache(b, h, cap, block, kind, fill=0):
    nb = -(-cap // block)
    k8, v8 = (torch.full((b, h, cap, HD), fill, dtype=torch.int8, device="cuda").view(KINDS[kind][0]) for _ in "kv")
    ks, vs = (torch.zeros((b, h, nb), device="cuda") for _ in "kv")
    return k8, v8, ks, vs


def snap(x, kind):
    """fp32 quotients to code values, half to even."""
    if kind == "int8":
        return np.clip(np.rint(np.nan_to_num(x)), -127, 127).astype(np.float32)
    return torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).float().numpy()


def define_write(codes, scales, x, pos, block, kind):
    """The definition on float32 code values [b][h][cap][64], scales [b][h][nb], tokens [b][n][h][64] fp16."""
    codes, scales = codes.copy(), scales.copy()
    b, h, cap, _ = codes.shape
    n, top = x.shape[1], np.float32(KINDS[kind][1])
    x = np.clip(x.astype(np.float32), -65504, 65504)
    with np.errstate(divide="ignore", invalid="ignore"):
        for i in range(b):
            p = int(pos[i])
            lo, hi = max(p, 0), min(p + n, cap)
            for g in range(h):
                for c in range(lo // block, -(-hi // block) if hi > lo else 0):
                    j0, j1 = max(lo, c * block), min(hi, (c + 1) * block)
                    part = x[i, j0 - p:j1 - p, g]
                    a = np.float32(np.nanmax(np.abs(part), initial=0.0))
                    s, old = a / top, scales[i, g, c]
                    if c * block < p:
                        s = max(s, old)
                    # the quotient by the unrounded scale, rounded to fp32
                    r = 1 / np.float64(s) if s != a / top else np.float64(top) / np.float64(a) if a > 0 else 0.0
                    if c * block < p and s != old:
                        codes[i, g, c * block:p] = snap((codes[i, g, c * block:p] * np.float64(old) * r).astype(np.float32), kind)
                    codes[i, g, j0:j1] = snap((part * r).astype(np.float32), kind)
                    scales[i, g, c] = s
    return codes, scales


def same_codes(t, want, kind):
    got = t.float().cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(got != want)[:5]


def tokens(gen, b, n, h, size=1.0):
    x = torch.randn((b, n, h, HD), generator=gen) * size * (0.1 + torch.rand((b, 1, h, 1), generator=gen))
    return x.to(torch.float16)


WRITES = [  # b, h, n, cap, positions (None: 0)
    (1, 1, 1, 1, None), (1, 1, 1, 16, [15]), (2, 3, 1, 40, [0, 39]), (3, 2, 5, 100, [14, 62, 98]), (1, 2, 100, 100, None),
    (4, 1, 33, 130, [-3, 0, 97, 120]), (2, 2, 1500, 1500, None), (3, 1, 2, 64, [64, -2, 1000]), (1, 20, 129, 448, [127]),
    (2, 2, 70, 50, [-30, 10]), (2, 1, 3, 50, [-2147483648, 2147483646])]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("case", WRITES)
def test_write_and_read(cuda, kind, block, case):
    b, h, n, cap, pos = case
    gen = torch.Generator().manual_seed(n * 7 + block)
    k8, v8, ks, vs = cache(b, h, cap, block, kind, fill=5)
    at = torch.tensor(pos, dtype=torch.int32) if pos else torch.zeros(b, dtype=torch.int32)
    # what the cache holds already: codes and scales of an earlier text
    for c8, s in ((k8, ks), (v8, vs)):
        c8.copy_((torch.randn(c8.shape, generator=gen) * 30).clamp(-120, 120).round().cuda().to(c8.dtype))
        s.copy_((torch.rand(s.shape, generator=gen) * 0.02).cuda())
    k, v = tokens(gen, b, n, h), tokens(gen, b, n, h, 3.0)
    want = [define_write(c8.float().cpu().numpy(), s.cpu().numpy(), x.numpy(), at.tolist(), block, kind)
            for c8, s, x in ((k8, ks, k), (v8, vs, v))]
    m.kv8_write(k.cuda(), v.cuda(), k8, v8, ks, vs, block=block, pos=at.cuda() if pos else None)
    torch.cuda.synchronize()
    for c8, s, (codes, scales) in ((k8, ks, want[0]), (v8, vs, want[1])):
        assert np.array_equal(s.cpu().numpy(), scales)
        same_codes(c8, codes, kind)
    # read them back: fp16 of the fp32 product code x scale
    kb, vb = (torch.full((b, n, h, HD), 7.0, dtype=torch.float16, device="cuda") for _ in "kv")
    lens = torch.tensor([cap - i for i in range(b)], dtype=torch.int32, device="cuda")
    m.kv8_read(k8, v8, ks, vs, kb, vb, block=block, pos=at.cuda(), lens=lens)
    for got, (codes, scales) in ((kb, want[0]), (vb, want[1])):
        val = codes * np.repeat(scales, block, 2)[:, :, :cap, None]
        ref = np.zeros((b, n, h, HD), np.float16)
        for i in range(b):
            for t in range(n):
                j = int(at[i]) + t
                if 0 <= j < cap - i:
                    ref[i, t] = val[i, :, j].astype(np.float16)
        assert np.array_equal(got.cpu().numpy(), ref)


@pytest.mark.parametrize("kind", list(KINDS))
def test_codes_at_the_border_between_two(cuda, kind):
    """New scales only: codes against x Q / a in whole numbers (products of fp16 values and Q, which 64 bits hold exactly),
    half to even. Some of the values lie exactly halfway between two codes; none may be a step off."""
    gen = torch.Generator().manual_seed(21)
    b, h, n, block = 4, 20, 1500, 64
    k8, v8, ks, vs = cache(b, h, n, block, kind)
    k = tokens(gen, b, n, h).cuda()
    m.kv8_write(k, k, k8, v8, ks, vs, block=block)
    x = torch.nn.functional.pad(k.double().transpose(1, 2), (0, 0, 0, -n % block)).view(b, h, -1, block, HD)
    a = x.abs().amax((3, 4), keepdim=True)
    top = KINDS[kind][1]
    # the step between codes there: 1, or an eighth of the power of two below the quotient (of at least 2^-6)
    if kind == "int8":
        step = torch.ones_like(x)
    else:
        powers = torch.tensor([2.0 ** i for i in range(-6, 9)], dtype=torch.float64, device="cuda")
        step = powers[(torch.searchsorted(powers, x.abs() * top / a, right=True) - 1).clamp(min=0)] / 8
    t = x.abs() * top / step  # exact: step is a power of two
    f = torch.floor(t / a)
    f = torch.where(f * a > t, f - 1, torch.where((f + 1) * a <= t, f + 1, f))
    rest = 2 * (t - f * a) - a
    up = (rest > 0) | ((rest == 0) & (f % 2 == 1))
    want = ((f + up) * step * x.sign()).view(b, h, -1, HD)[:, :, :n]
    assert (rest == 0).sum() > (100 if kind == "int8" else 1000)
    assert torch.equal(k8.double(), want) and torch.equal(v8.double(), want)


@pytest.mark.parametrize("kind", list(KINDS))
def test_write_zero_infinite_and_nan(cuda, kind):
    k = torch.zeros((1, 64, 1, HD), dtype=torch.float16)
    k[0, 16, 0, 3] = float("inf")
    k[0, 17, 0, 4] = float("-inf")
    k[0, 18, 0, 5] = 2.0
    k[0, 33, 0, 6] = float("nan")
    k[0, 34, 0, 7] = 1.5
    k[0, 50, 0, 8] = 6e-8  # the smallest fp16 number
    k8, v8, ks, vs = cache(1, 1, 64, 16, kind)
    m.kv8_write(k.cuda(), k.cuda(), k8, v8, ks, vs, block=16)
    top = np.float32(KINDS[kind][1])
    want = np.array([0, 65504, 1.5, np.float32(np.float16(6e-8))], np.float32) / top
    assert np.array_equal(ks.cpu().numpy()[0, 0], want) and torch.equal(ks, vs)
    c = k8.float().cpu().numpy()[0, 0]
    assert c[16, 3] == top and c[17, 4] == -top and c[34, 7] == top and c[50, 8] == top
    assert not c[:16].any() and (c[33, 6] == 0 if kind == "int8" else np.isnan(c[33, 6]))
    codes, _ = define_write(np.zeros((1, 1, 64, HD), np.float32), np.zeros((1, 1, 4), np.float32), k.numpy(), [0], 16, kind)
    same_codes(k8, codes, kind)
    same_codes(v8, codes, kind)


@pytest.mark.parametrize("kind", list(KINDS))
def test_tokens_one_by_one_stay_within_their_steps(cuda, kind):
    """A text written token by token: a code is rounded again each time its block's scale grows, so a value is off by at
    most half a step of every scale it has been on; those scales are below the last one, and the number of times a
    running maximum of 32 x 64 values grows is counted."""
    gen = torch.Generator().manual_seed(3)
    b, h, cap, block = 2, 2, 70, 32
    k8, v8, ks, vs = cache(b, h, cap, block, kind)
    k, v = tokens(gen, b, cap, h), tokens(gen, b, cap, h)
    kd, vd = k.cuda(), v.cuda()
    pos = torch.zeros(b, dtype=torch.int32, device="cuda")
    for t in range(cap):
        m.kv8_write(kd[:, t:t + 1], vd[:, t:t + 1], k8, v8, ks, vs, block=block, pos=pos)
        pos += 1
    x = k.float().numpy().transpose(0, 2, 1, 3)
    got = (k8.float() * ks.repeat_interleave(block, 2)[:, :, :cap, None]).cpu().numpy()
    for i in range(b):
        for g in range(h):
            for c in range(-(-cap // block)):
                part = x[i, g, c * block:(c + 1) * block]
                s = ks[i, g, c].item()
                assert np.float32(np.abs(part).max()) / np.float32(KINDS[kind][1]) == np.float32(s)
                tops = np.maximum.accumulate(np.abs(part).max(1))
                grown = 1 + int((np.diff(tops) > 0).sum())
                if kind == "int8":
                    step = np.full_like(part, s / 2)
                else:  # half a step: 2^-4 of the value, of at least the smallest normal code's, 2^-6
                    step = np.maximum(np.abs(part) * (1 + grown * 2.0 ** -4), 2.0 ** -6 * s) * 2.0 ** -4
                err = np.abs(got[i, g, c * block:(c + 1) * block] - part)
                assert (err <= grown * step * (1 + 2.0 ** -20)).all()


def attend_ref(q, k, v, lens, causal, scale=0.125):
    """64-bit out [b][rows][hq][64] and probs [b][hq][rows][cap] of values k, v [b][hkv][cap][64], and the tolerances."""
    b, rows, hq, _ = q.shape
    hkv, cap = k.shape[1], k.shape[2]
    out, tol = np.zeros((b, rows, hq, HD)), np.zeros((b, rows, hq, 1))
    p, ptol = np.zeros((b, hq, rows, cap)), np.zeros((b, hq, rows, 1))
    for i in range(b):
        n = max(0, min(int(lens[i]), cap))
        for hh in range(hq):
            g = hh // (hq // hkv)
            for r in range(rows):
                lim = max(0, n - rows + r + 1) if causal else n
                if not lim:
                    continue
                kk, vv, qq = k[i, g, :lim], v[i, g, :lim], q[i, r, hh]
                s = kk @ qq * scale
                e = np.exp(s - s.max())
                w = e / e.sum()
                big = (np.abs(kk) @ np.abs(qq)).max() * scale
                rel = 4 * 2.0 ** -16 * big + 2.0 ** -20 + (lim / 4 + 64) * 2.0 ** -23
                p[i, hh, r, :lim], ptol[i, hh, r] = w, rel
                out[i, r, hh], tol[i, r, hh] = w @ vv, 2 * rel * np.abs(vv).max()
    return out, tol, p, ptol


def check(got, want, tol):
    got = got.float().cpu().numpy().astype(np.float64)
    lim = np.abs(want) * 2.0 ** -11 + 2.0 ** -25 + tol
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > lim
    assert not bad.any(), (np.argwhere(bad)[:4], (np.abs(got - want) / lim).max())


def filled(gen, b, h, cap, block, kind):
    k8, v8, ks, vs = cache(b, h, cap, block, kind)
    for c8, s in ((k8, ks), (v8, vs)):
        x = torch.randn(c8.shape, generator=gen) * (36 if kind == "int8" else 120)
        c8.copy_((x.round().clamp(-127, 127) if kind == "int8" else x.clamp(-448, 448)).cuda().to(c8.dtype))
        s.copy_(((0.2 + torch.rand(s.shape, generator=gen)) / (36 if kind == "int8" else 120)).cuda())
    return k8, v8, ks, vs


def values(c8, s, block):
    return (c8.double() * s.double().repeat_interleave(block, 2)[:, :, :c8.shape[2], None]).cpu().numpy()


ATTENDS = [  # b, rows, kv heads, group, cap, lens (None: cap), causal
    (1, 1, 1, 1, 1, None, False), (2, 1, 6, 1, 1500, None, False), (3, 1, 2, 1, 64, [0, 1, 64], False),
    (2, 1, 1, 4, 200, [199, 65], False), (1, 5, 3, 1, 1500, None, False), (2, 7, 2, 2, 97, [97, 33], True),
    (3, 40, 2, 1, 70, [70, 40, 11], True), (1, 223, 1, 1, 448, None, True), (1, 33, 1, 3, 130, [129], False),
    (2, 3, 1, 1, 2, [1, 2], True), (1, 1, 1, 1, 20000, None, False), (4, 1, 20, 1, 448, [17, 448, 15, 16], False),
    (2, 1, 3, 1, 33, [-5, 1000000], False), (1, 9, 1, 8, 300, [300], True), (150, 1, 8, 1, 100, None, False),
    # many chunks: an equal share of them to each warp, whatever the lengths
    (32, 1, 20, 1, 448, [14 * i for i in range(32)], False), (2, 1, 4, 2, 30000, [30000, 17], False),
    (40, 3, 16, 1, 400, [(37 * i) % 401 for i in range(40)], True), (4, 2, 8, 4, 8000, [8000, 1, 0, 7999], True),
    (64, 1, 16, 1, 300, [i % 3 * 32 for i in range(64)], False), (60, 1, 20, 1, 200, [0] * 60, False),
    (100, 1, 12, 1, 257, [200 + i % 58 for i in range(100)], False), (1, 8, 1, 1, 230000, None, True),
    # tiles of 16 rows, more than two to an SM
    (25, 20, 6, 1, 448, [18 * i + 16 for i in range(25)], True), (10, 11, 13, 3, 400, [40 * i for i in range(10)], True),
    (40, 9, 8, 1, 300, [300 - i for i in range(40)], False),
    # prompts that fill the GPU: each warp takes rows of its own
    (38, 37, 8, 1, 150, [4 * i - 1 for i in range(38)], True), (40, 11, 8, 3, 90, [(29 * i) % 91 for i in range(40)], True),
    (45, 17, 10, 1, 65, [63 + i % 3 for i in range(45)], False), (30, 33, 10, 1, 128, None, True)]


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("case", ATTENDS, ids=lambda c: "x".join(map(str, c[:5])))
def test_attention(cuda, kind, block, case):
    b, rows, h, group, cap, lens, causal = case
    gen = torch.Generator().manual_seed(cap + block)
    hq = h * group
    c = filled(gen, b, h, cap, block, kind)
    q = (torch.randn((b, rows, hq, HD), generator=gen) * 1.5).to(torch.float16)
    ln = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    out = torch.full((b, rows, hq, HD), 9.0, dtype=torch.float16, device="cuda")
    pslot = torch.full((hq,), -1, dtype=torch.int32)
    pslot[hq - 1] = 0
    if hq > 1:
        pslot[0] = 1
    slots = min(2, hq)
    probs = torch.full((b, slots, rows, cap), 9.0, dtype=torch.float16, device="cuda")
    m.attn8(q.cuda(), *c, out, block=block, lens=None if ln is None else ln.cuda(), causal=causal, probs=probs,
            pslot=pslot.cuda())
    torch.cuda.synchronize()
    k, v = values(c[0], c[2], block), values(c[1], c[3], block)
    want, tol, p, ptol = attend_ref(q.double().numpy(), k, v, [cap] * b if lens is None else lens, causal)
    check(out, want, tol)
    for hh in range(hq):
        if pslot[hh] >= 0:
            check(probs[:, pslot[hh]], p[:, hh], ptol[:, hh] * p[:, hh])
    # the same without probabilities
    again = torch.full_like(out, 3.0)
    m.attn8(q.cuda(), *c, again, block=block, lens=None if ln is None else ln.cuda(), causal=causal)
    check(again, want, tol)
    assert m.status()[0] == 0


@pytest.mark.parametrize("rows,h", [(1, 2), (20, 2), (20, 230)])
def test_nan_behind_the_sequence_is_not_used(cuda, rows, h):
    gen = torch.Generator().manual_seed(1)
    b, cap, block = 2, 150, 32
    c = filled(gen, b, h, cap, block, "e4m3")
    lens = [70, 0]
    for x in c[:2]:
        x.view(torch.int8)[0, :, 70:] = 0x7f
        x.view(torch.int8)[1] = 0x7f
    for s in c[2:]:
        s[0, :, 3:] = float("nan")
        s[1] = float("inf")
    q = torch.randn((b, rows, h, HD), generator=gen).to(torch.float16)
    out = torch.empty((b, rows, h, HD), dtype=torch.float16, device="cuda")
    probs = torch.empty((b, 1, rows, cap), dtype=torch.float16, device="cuda")
    m.attn8(q.cuda(), *c, out, block=block, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), probs=probs,
            pslot=torch.tensor([-1, 0] + [-1] * (h - 2), dtype=torch.int32, device="cuda"))
    k, v = (np.nan_to_num(values(x, s, block)) for x, s in ((c[0], c[2]), (c[1], c[3])))
    want, tol, p, ptol = attend_ref(q.double().numpy(), k, v, lens, False)
    check(out, want, tol)
    check(probs[:, 0], p[:, 1], ptol[:, 1] * p[:, 1])


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rows,block,heads,bad", [
    (4, 16, 2, "nan"), (6, 16, 2, "inf"), (40, 16, 2, "nan"), (40, 32, 2, "inf"), (130, 64, 2, "nan"), (40, 16, 300, "nan"),
    (130, 64, 100, "inf")])
def test_scales_that_are_not_finite_reach_only_the_rows_that_see_them(cuda, kind, rows, block, heads, bad):
    """Causal rows over one sequence; the scales of the block that ends the sequence are NaN or infinite. The rows before
    it come out bit for bit as with a finite scale there, those that see it are NaN."""
    gen = torch.Generator().manual_seed(rows)
    L = 3 * block + 1 if rows < block else rows + 1  # the last block starts inside the rows
    cap = -(-L // block) * block
    last = (L - 1) // block
    k8, v8, ks, vs = cache(1, heads, cap, block, kind)
    for c8, s in ((k8, ks), (v8, vs)):
        c8.copy_((torch.randn(c8.shape, generator=gen) * 30).clamp(-120, 120).round().cuda().to(c8.dtype))
        s.copy_((0.001 + torch.rand(s.shape, generator=gen) * 0.02).cuda())
    q = torch.randn((1, rows, heads, HD), generator=gen).half().cuda()
    lens = torch.tensor([L], dtype=torch.int32, device="cuda")
    out, want = torch.empty_like(q), torch.empty_like(q)
    m.attn8(q, k8, v8, ks, vs, want, block=block, lens=lens, causal=True)
    sees = L - rows + 1 + torch.arange(rows, device="cuda") > last * block
    assert sees.any() and not sees.all()
    for s in (vs, ks):
        keep = s[:, :, last].clone()
        s[:, :, last] = float(bad)
        m.attn8(q, k8, v8, ks, vs, out, block=block, lens=lens, causal=True)
        s[:, :, last] = keep
        assert torch.equal(out[0, ~sees], want[0, ~sees])
        if s is vs or bad == "nan":
            assert out[0, sees].isnan().all()


def test_large_and_small_scores(cuda):
    """Scores far apart: one position holds all the weight, then none does (equal scores)."""
    b, h, cap, block = 1, 1, 300, 64
    for kind, big in (("int8", 127), ("e4m3", 448)):
        k8, v8, ks, vs = cache(b, h, cap, block, kind)
        gen = torch.Generator().manual_seed(2)
        ks.fill_(100.0)
        vs.fill_(0.01)
        v8.copy_(torch.randint(-100, 100, v8.shape, generator=gen).cuda().to(v8.dtype))
        v = values(v8, vs, block)[0, 0]
        q = torch.full((1, 1, 1, HD), 50.0, dtype=torch.float16, device="cuda")
        out = torch.empty_like(q)
        m.attn8(q, k8, v8, ks, vs, out, block=block)  # all scores 0: the mean
        check(out[0, 0], v.mean(0, keepdims=True), (cap / 4 + 64) * 2.0 ** -22 * np.abs(v).max())
        k8.view(torch.int8)[0, 0, 211] = 127 if kind == "int8" else 0x7e
        m.attn8(q, k8, v8, ks, vs, out, block=block)
        check(out[0, 0], v[211:212], 2.0 ** -20)
        k8.view(torch.int8)[0, 0] = -127 if kind == "int8" else -2  # all scores equal and very low
        m.attn8(q, k8, v8, ks, vs, out, block=block)
        # equal scores, computed alike: the weights are equal whatever their rounding
        check(out[0, 0], v.mean(0, keepdims=True), (cap / 4 + 64) * 2.0 ** -22 * np.abs(v).max())


def test_strides_of_the_engine_and_of_a_projection(cuda):
    """The cache as one layer of [sequence][layer][k|v][head][position], q, k, v as slices of one projection."""
    gen = torch.Generator().manual_seed(4)
    b, nl, h, cap, block = 3, 2, 4, 90, 32
    codes = torch.zeros((b, nl, 2, h, cap, HD), dtype=torch.int8, device="cuda")
    scales = torch.zeros((b, nl, 2, h, 3), device="cuda")
    qkv = torch.randn((b, 50, 3 * h, HD), generator=gen).to(torch.float16).cuda()
    q, k, v = qkv[:, :, :h], qkv[:, :, h:2 * h], qkv[:, :, 2 * h:]
    c = (codes[:, 1, 0], codes[:, 1, 1], scales[:, 1, 0], scales[:, 1, 1])
    m.kv8_write(k, v, *c, block=block, pos=torch.full((b,), 40, dtype=torch.int32, device="cuda"))
    assert not codes[:, 0].any() and not scales[:, 0].any()
    codes2 = np.zeros((b, h, cap, HD), np.float32)
    want, sc = define_write(codes2, np.zeros((b, h, 3), np.float32), k.cpu().numpy(), [40] * b, block, "int8")
    same_codes(c[0], want, "int8")
    big = torch.full((b, 50, 2 * h, HD), 5.0, dtype=torch.float16, device="cuda")
    m.attn8(q, *c, big[:, :, h:], block=block, causal=True)
    assert (big[:, :, :h] == 5).all()
    kk, vv = (values(x.contiguous(), s.contiguous(), block) for x, s in ((c[0], c[2]), (c[1], c[3])))
    ref, tol, _, _ = attend_ref(q.double().cpu().numpy(), kk, vv, [cap] * b, True)
    check(big[:, :, h:], ref, tol)
    kb = torch.empty((b, 50, 3, h, HD), dtype=torch.float16, device="cuda")
    m.kv8_read(*c, kb[:, :, 0], kb[:, :, 2], block=block, pos=torch.full((b,), 40, dtype=torch.int32, device="cuda"))
    assert np.array_equal(kb[:, :, 0].cpu().numpy(), (want * np.repeat(sc, block, 2)[:, :, :cap, None])[
        :, :, 40:].transpose(0, 2, 1, 3).astype(np.float16))


def test_offsets_past_32_bits(cuda):
    """A head of 2^25 + 20 positions (more than 2^31 bytes of keys): the last one holds the weight."""
    cap, block = (1 << 25) + 20, 128
    k8, v8, ks, vs = cache(1, 1, cap, block, "int8")
    k = torch.full((1, 20, 1, HD), 8.0, dtype=torch.float16, device="cuda")
    v = torch.arange(20, device="cuda").half()[None, :, None, None].expand(1, 20, 1, HD).contiguous()
    k[0, :19] = 0
    pos = torch.tensor([1 << 25], dtype=torch.int32, device="cuda")
    m.kv8_write(k, v, k8, v8, ks, vs, block=block, pos=pos)
    q = torch.full((1, 1, 1, HD), 8.0, dtype=torch.float16, device="cuda")  # its score is 512, the others' 0
    out = torch.empty_like(q)
    m.attn8(q, k8, v8, ks, vs, out, block=block)
    assert (out == 19).all()
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    m.kv8_read(k8, v8, ks, vs, kb, vb, block=block, pos=pos)
    assert (kb[0, 19] == 8).all() and (kb[0, :19] == 0).all() and (vb[0, 19] == 19).all()


def test_decoding_in_a_graph_and_on_two_streams(cuda):
    """Write a token and attend, captured once and replayed along the sequence, against eager calls; two such graphs on
    two streams with scratch of their own."""
    gen = torch.Generator().manual_seed(6)
    b, h, cap, block, steps = 2, 3, 200, 32, 40
    tok = [torch.randn((2, steps, b, 1, 3 * h, HD), generator=gen).to(torch.float16).cuda() for _ in "ab"]
    eager = []
    sides = []
    for i in range(2):
        for mode in ("eager", "graph"):
            kind = ("int8", "e4m3")[i]
            c = cache(b, h, cap, block, kind)
            pos = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
            lens = pos + 1
            qkv = torch.empty((b, 1, 3 * h, HD), dtype=torch.float16, device="cuda")
            out = torch.empty((b, 1, h, HD), dtype=torch.float16, device="cuda")
            need = m.attn8_scratch_bytes(b, 1, h, h, cap)
            scratch = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")

            def step(c=c, pos=pos, lens=lens, qkv=qkv, out=out, scratch=scratch):
                m.kv8_write(qkv[:, :, h:2 * h], qkv[:, :, 2 * h:], *c, block=block, pos=pos)
                m.attn8(qkv[:, :, :h], *c, out, block=block, lens=lens, scratch=scratch)
                pos.add_(1)
                lens.add_(1)

            if mode == "eager":
                outs = []
                for t in range(steps):
                    qkv.copy_(tok[i][0, t])
                    step()
                    outs.append(out.clone())
                eager.append((outs, [x.clone() for x in c]))
            else:
                st = torch.cuda.Stream()
                g = torch.cuda.CUDAGraph()
                st.wait_stream(torch.cuda.current_stream())
                with torch.cuda.graph(g, stream=st):
                    step()
                sides.append((g, st, qkv, out, c, i, (pos, lens, scratch)))  # a graph keeps no tensor alive
    torch.cuda.synchronize()
    got = [[], []]
    for t in range(steps):
        for g, st, qkv, out, c, i, _ in sides:
            with torch.cuda.stream(st):
                qkv.copy_(tok[i][0, t])
                g.replay()
                got[i].append(out.clone())
    torch.cuda.synchronize()
    for g, st, qkv, out, c, i, _ in sides:
        assert all(torch.equal(x, y) for x, y in zip(got[i], eager[i][0]))
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(c, eager[i][1]))


def test_sequences_that_share_a_cache(cuda):
    """Several sequences over one cache (a sequence stride of 0), each with its own length; odd strides of dimensions of
    one."""
    gen = torch.Generator().manual_seed(8)
    b, h, cap, block = 5, 3, 150, 32
    c = filled(gen, 1, h, cap, block, "int8")
    shared = [x.expand(b, *x.shape[1:]) for x in c]
    lens = torch.tensor([1, 150, 33, 0, 64], dtype=torch.int32)
    q = torch.randn((b, 1, h, HD), generator=gen).to(torch.float16)
    out = torch.empty_like(q, device="cuda")
    m.attn8(q.cuda(), *shared, out, block=block, lens=lens.cuda())
    k, v = (np.repeat(values(x, s, block), b, 0) for x, s in ((c[0], c[2]), (c[1], c[3])))
    want, tol, _, _ = attend_ref(q.double().numpy(), k, v, lens.tolist(), False)
    check(out, want, tol)
    with pytest.raises(m.MmzError, match="overlap"):
        m.kv8_write(out, out, *shared, block=block)
    one = torch.empty((1, 3, h, HD), dtype=torch.float16, device="cuda").as_strided((1, 1, h, HD), (7, 13, HD, 1))
    one.copy_(q[:1].cuda())
    o1 = torch.empty((1, 1, h, HD), dtype=torch.float16, device="cuda").as_strided((1, 1, h, HD), (3, 5, HD, 1))
    m.attn8(one, *c, o1, block=block, lens=lens[:1].cuda())
    assert torch.equal(o1, out[:1])


def test_scratch_of_a_call_on_another_stream(cuda):
    """Calls without scratch on a stream that is not the current one, while the current one allocates and writes."""
    gen = torch.Generator().manual_seed(9)
    c = filled(gen, 1, 2, 60000, 64, "int8")
    q = torch.randn((1, 1, 2, HD), generator=gen).to(torch.float16).cuda()
    want = torch.empty_like(q)
    assert m.attn8_scratch_bytes(1, 1, 2, 2, 60000) > 0
    m.attn8(q, *c, want, block=64)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    outs = [torch.empty_like(q) for _ in range(20)]
    for i, out in enumerate(outs):
        m.attn8(q, *c, out, block=64, stream=st if i % 2 else st.cuda_stream)
        torch.full((m.attn8_scratch_bytes(1, 1, 2, 2, 60000),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("raw", [False, True])
def test_scratch_is_no_memory_of_the_current_stream(cuda, raw):
    """A freed tensor of the scratch's size that the current stream has yet to read, and calls without scratch on both
    streams in turn, nobody waiting: each call's scratch is memory of the stream it runs on."""
    gen = torch.Generator().manual_seed(19)
    caches = [filled(gen, 1, 2, 60000, 64, "int8") for _ in "ab"]
    q = torch.randn((1, 1, 2, HD), generator=gen).to(torch.float16).cuda()
    need = m.attn8_scratch_bytes(1, 1, 2, 2, 60000)
    assert need > 0
    want = [torch.empty_like(q) for _ in "ab"]
    for c, w in zip(caches, want):
        m.attn8(q, *c, w, block=64)
    st = torch.cuda.Stream()
    on = st.cuda_stream if raw else st
    outs = [torch.zeros_like(q) for _ in range(41)]
    held = torch.full((need,), 7, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(100000000)  # some 50 ms on the current stream
    read = held.clone()
    del held  # its block is free for the current stream, behind the copy
    m.attn8(q, *caches[0], outs[40], block=64, stream=on)
    for i in range(0, 40, 2):
        m.attn8(q, *caches[0], outs[i], block=64)
        m.attn8(q, *caches[1], outs[i + 1], block=64, stream=on)
    torch.cuda.synchronize()
    assert (read == 7).all()
    assert all(torch.equal(out, want[i & 1]) for i, out in enumerate(outs))


def test_captured_calls_without_scratch(cuda):
    """Calls that allocate their scratch inside a capture, on the captured stream and on one that joins it, replayed beside
    eager calls and those of two threads on streams of their own; the default stream by number."""
    import threading
    gen = torch.Generator().manual_seed(22)
    caches = [filled(gen, 1, 2, 60000, 64, "int8") for _ in range(3)]
    q = torch.randn((1, 1, 2, HD), generator=gen).to(torch.float16).cuda()
    assert m.attn8_scratch_bytes(1, 1, 2, 2, 60000) > 0
    want = [torch.empty_like(q) for _ in caches]
    for c, w in zip(caches, want):
        m.attn8(q, *c, w, block=64, stream=0)
    torch.cuda.synchronize()
    outs = [torch.zeros_like(q) for _ in caches]
    st, other, g = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        other.wait_stream(st)
        m.attn8(q, *caches[0], outs[0], block=64)
        m.attn8(q, *caches[1], outs[1], block=64, stream=other)
        m.attn8(q, *caches[2], outs[2], block=64)
        st.wait_stream(other)
    eager = [[torch.zeros_like(q) for _ in range(20)] for _ in range(3)]

    def calls(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for out in eager[k]:
                m.attn8(q, *caches[k], out, block=64)

    threads = [threading.Thread(target=calls, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for out in eager[2]:
        g.replay()
        m.attn8(q, *caches[2], out, block=64)
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    assert all(torch.equal(out, w) for outs3, w in zip(eager, want) for out in outs3)


def test_strides_of_dimensions_of_one_may_differ(cuda):
    """One token: keys [b][n][h][64], values head by head and transposed; a cache of one sequence, one head and one block
    whose values and scales come from larger tensors."""
    gen = torch.Generator().manual_seed(20)
    b, h, cap, block = 2, 3, 40, 32
    k = tokens(gen, b, 1, h).cuda()
    v = tokens(gen, b, 1, h).cuda()
    vt = torch.empty((b, h, 1, HD), dtype=torch.float16, device="cuda").transpose(1, 2).copy_(v)
    assert vt.stride() == (h * HD, HD, HD, 1) != k.stride()
    a, c = cache(b, h, cap, block, "int8"), cache(b, h, cap, block, "int8")
    pos = torch.tensor([0, 33], dtype=torch.int32, device="cuda")
    m.kv8_write(k, v, *a, block=block, pos=pos)
    m.kv8_write(k, vt, *c, block=block, pos=pos)
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    kb, vb = torch.empty_like(k), torch.empty((b, h, 1, HD), dtype=torch.float16, device="cuda").transpose(1, 2)
    want = torch.empty_like(k), torch.empty_like(k)
    m.kv8_read(*c, kb, vb, block=block, pos=pos)
    m.kv8_read(*c, *want, block=block, pos=pos)
    assert torch.equal(kb, want[0]) and torch.equal(vb, want[1])
    small, wide = filled(gen, 1, 1, 20, block, "int8"), cache(4, 5, 20, block, "int8")
    for x, y in zip(small, wide):
        y[2:3, 3:4] = x
    q = torch.randn((1, 1, 2, HD), generator=gen).half().cuda()
    one, two = torch.empty_like(q), torch.empty_like(q)
    m.attn8(q, *small, one, block=block)
    m.attn8(q, small[0], wide[1][2:3, 3:4], small[2], wide[3][2:3, 3:4], two, block=block)
    assert torch.equal(one, two)
    with pytest.raises(m.MmzError, match="same strides"):
        m.kv8_write(k, v[:, :, :1].expand(b, 1, h, HD), *a, block=block)


@pytest.mark.parametrize("b,rows,h,group,cap,causal", [
    (2, 1, 3, 1, 1500, False), (1, 1, 2, 4, 60000, False), (3, 7, 2, 1, 400, True), (2, 30, 4, 1, 200, True),
    (40, 20, 8, 1, 448, True), (40, 37, 8, 1, 150, True), (1, 2, 1, 8, 9000, False)])
def test_the_output_in_place_of_the_queries(cuda, b, rows, h, group, cap, causal):
    """out as q itself, and beside it in one tensor: the same bits as apart from it, whatever the layout of the call."""
    gen = torch.Generator().manual_seed(cap)
    c = filled(gen, b, h, cap, 64, "int8")
    lens = torch.tensor([cap - 5 * i for i in range(b)], dtype=torch.int32, device="cuda")
    hq = h * group
    q = torch.randn((b, rows, hq, HD), generator=gen).half().cuda()
    want = torch.empty_like(q)
    m.attn8(q, *c, want, block=64, lens=lens, causal=causal)
    both = torch.zeros((b, rows, 2, hq, HD), dtype=torch.float16, device="cuda")
    both[:, :, 1] = q
    m.attn8(both[:, :, 1], *c, both[:, :, 0], block=64, lens=lens, causal=causal)
    assert torch.equal(both[:, :, 0], want) and torch.equal(both[:, :, 1], q)
    same = q.clone()
    m.attn8(same, *c, same, block=64, lens=lens, causal=causal)
    assert torch.equal(same, want)
    with pytest.raises(m.MmzError, match="out over q"):
        m.attn8(both.view(b, rows, 2 * hq, HD)[:, :, 1:hq + 1], *c, both[:, :, 0], block=64, lens=lens, causal=causal)


def test_refusals(cuda):
    c = cache(1, 2, 64, 32, "int8")
    q = torch.zeros((1, 1, 2, HD), dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    lens = torch.ones(1, dtype=torch.int32, device="cuda")
    bad = [lambda: m.attn8(q.float(), *c, out, block=32), lambda: m.attn8(q, *c, out[:, :, :1], block=32),
           lambda: m.attn8(q, *c, out, block=64), lambda: m.attn8(q, *c, out, block=32, lens=lens.long()),
           lambda: m.attn8(q, *c, out, block=32, lens=lens.expand(2)), lambda: m.attn8(q[:, :, :1], *c, out, block=32),
           lambda: m.attn8(q.cpu(), *c, out, block=32), lambda: m.attn8(q, c[0], c[1].transpose(1, 2), *c[2:], out, block=32),
           lambda: m.attn8(q, *c, out, block=32, probs=torch.empty((1, 1, 1, 63), dtype=torch.float16, device="cuda"),
                           pslot=torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: m.attn8(q, *c, out, block=32, probs=torch.empty((1, 1, 1, 64), dtype=torch.float16, device="cuda")),
           lambda: m.attn8(q, q, q, *c[2:], out, block=32), lambda: m.attn8(q, *c, out, block=20),
           lambda: m.kv8_write(q, q[:, :, :1], *c, block=32), lambda: m.kv8_write(q, q, *c, block=32, pos=lens.float()),
           lambda: m.kv8_read(*c, q, q.float(), block=32)]
    for call in bad:
        with pytest.raises(m.MmzError):
            call()
    with pytest.raises(m.MmzError, match="multiple of kv_heads"):
        m.attn8(q[:, :, :1], *c, out[:, :, :1], block=32)
    e = torch.empty((0, 1, 2, HD), dtype=torch.float16, device="cuda")
    m.attn8(e, *(x[:0] for x in c), torch.empty_like(e), block=32)  # no sequences: nothing to do
