"""Token log probabilities on the GPU against 64 bits.

Tolerances: an exponential is off by at most 2^-21 of its value (argument and approximation); a row's sum of V positive
terms by (V / 256 + 64) 2^-23 (partial sums of at most V / 256 terms in a row, then joined) and 2^-20 for the joins'
exponentials; so log sum is off by E = (V / 256 + 64) 2^-23 + 2^-19, lse and a log probability by E plus an fp32 step of
the largest number involved. The entropy's second sum has terms e^d |d|: E times (1 + their weighted mean), taken with
the mean of |d| from the 64-bit row. For hidden states, the products' sums are exact (operands on a grid), as in fp32.
"""
import ctypes

import numpy as np
import pytest
import torch
from test_serving_args import Logprobs

import mimizuku_b200 as m

pytestmark = pytest.mark.gpu


def reference(x, target, sup, top):
    """64-bit values of one batch of logits [rows][V] (float64 numpy), and the tolerances of lse / logp and entropy."""
    rows, V = x.shape
    x = x.copy()
    if sup is not None:
        x[:, sup != 0] = -np.inf
    mx = x.max(1)
    some = mx > -np.inf
    d = x - np.where(some, mx, 0)[:, None]
    e = np.exp(d)
    s = e.sum(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        lse = np.where(some, mx + np.log(s), -np.inf)
        mean = np.where(some, (e * np.where(e > 0, d, 0)).sum(1) / s, 0)
        ent = np.where(some, np.log(s) - mean, 0)
        ok = (target >= 0) & (target < V)
        xt = x[np.arange(rows), np.where(ok, target, 0)]
        logp = np.where(ok, np.where(xt == -np.inf, -np.inf, xt - lse), 0)
    ids, tlp = np.full((rows, top), -1), np.full((rows, top), -np.inf)
    for r in range(rows):
        order = np.argsort(-x[r], kind="stable")[:top]
        order = order[x[r, order] > -np.inf]
        ids[r, :len(order)], tlp[r, :len(order)] = order, x[r, order] - lse[r]
    E = (V / 256 + 64) * 2.0 ** -23 + 2.0 ** -19
    big = np.where(some, np.abs(mx), 0) + np.log(np.maximum(s, 1))
    return dict(lse=lse, entropy=ent, logp=logp, top_id=ids, top_logp=tlp), E + big * 2.0 ** -22, 2 * E * (1 + np.abs(mean))


def buffers(rows, top):
    z = lambda *s: torch.full(s, 77.0, device="cuda")  # noqa: E731
    return dict(logp=z(rows), entropy=z(rows), lse=z(rows),
                top_id=torch.full((rows, top), 77, dtype=torch.int32, device="cuda") if top else None,
                top_logp=z(rows, top) if top else None)


def near(got, want, tol):
    got = got.double().cpu().numpy()
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    tol = np.broadcast_to(tol, want.shape)
    bad = ~(np.abs(got[~inf] - want[~inf]) <= tol[~inf] + np.abs(want[~inf]) * 2.0 ** -23)
    assert not bad.any(), (got[~inf][bad][:4], want[~inf][bad][:4], tol[~inf][bad][:4])


def compare(o, ref, top):
    want, tol, etol = ref
    torch.cuda.synchronize()
    if top:
        assert np.array_equal(o["top_id"].cpu().numpy(), want["top_id"])
        near(o["top_logp"], want["top_logp"], tol[:, None] + np.abs(np.where(np.isinf(want["top_logp"]), 0, want[
            "top_logp"])) * 2.0 ** -22)
    near(o["lse"], want["lse"], tol)
    near(o["logp"], want["logp"], tol + np.where(np.isinf(want["logp"]), 0, np.abs(want["logp"])) * 2.0 ** -22)
    near(o["entropy"], want["entropy"], etol)


SHAPES = [(1, 1, 1), (3, 2, 2), (2, 7, 8), (5, 31, 3), (4, 33, 0), (2, 300, 8), (1, 4097, 5), (7, 51865, 5), (3, 51866, 8),
          (40, 1000, 4), (2, 131075, 5), (300, 513, 1), (600, 2048, 5)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("masked", [False, True])
def test_rows_of_logits(cuda, dtype, shape, masked):
    rows, V, top = shape
    gen = torch.Generator().manual_seed(V)
    x = (torch.randn((rows, V + 3), generator=gen) * 3).to(dtype)[:, :V]  # a row pitch that is not the vocabulary
    target = torch.randint(-1, V + 1, (rows,), generator=gen, dtype=torch.int32)
    sup = None
    if masked:
        sup = (torch.rand(V, generator=gen) < 0.3).to(torch.uint8)
    o = buffers(rows, top)
    xd = torch.empty((rows, V + 3), dtype=dtype, device="cuda")[:, :V]
    xd.copy_(x)
    m.token_logprobs(xd, target.cuda(), **o, sup=None if sup is None else sup.cuda())
    compare(o, reference(x.double().numpy(), target.numpy(), None if sup is None else sup.numpy(), top), top)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [5, 999, 51866])
def test_rows_with_ties_and_infinities(cuda, dtype, V):
    """Constant rows, rows of few values, rows of -inf with a few finite logits, a row of -inf only, the type's lowest
    value as a mask, one logit far above the rest."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randint(-2, 3, (10, V), generator=gen).to(dtype)
    x[1] = 3.5
    x[2] = -float("inf")
    x[2, [1, V - 1]] = torch.tensor([2.0, 5.0], dtype=dtype)
    x[3] = -float("inf")
    x[4] = torch.finfo(dtype).min
    x[4, V // 2] = 1.0
    x[5] = -20000.0
    x[5, 3] = 20000.0
    x[6] = torch.arange(V).to(dtype) / V
    x[7] = -torch.arange(V).to(dtype) / V
    x[8] = 0.0
    x[8, ::2] = -0.0
    x[9] = torch.finfo(dtype).min
    target = torch.tensor([0, V - 1, 1, 2, 0, 3, V - 1, V, -1, 2], dtype=torch.int32)
    o = buffers(10, 8)
    m.token_logprobs(x.cuda(), target.cuda(), **o)
    compare(o, reference(x.double().numpy(), target.numpy(), None, 8), 8)


def test_nan_and_plus_infinity(cuda):
    x = torch.randn((4, 700))
    x[0, 5] = float("nan")
    x[1, 6] = float("inf")
    x[2, 7] = float("nan")
    sup = torch.zeros(700, dtype=torch.uint8)
    sup[7] = 1  # a suppressed NaN is not read into anything
    x[0, 7] = x[1, 7] = 0.5
    o = buffers(4, 3)
    target = torch.tensor([1, 2, 3, 4], dtype=torch.int32)
    m.token_logprobs(x.cuda(), target.cuda(), **o, sup=sup.cuda())
    for n in ("lse", "logp", "entropy"):
        assert torch.isnan(o[n]).tolist() == [True, True, False, False], n
    y = x[2:].clone()
    y[:, 7] = 0
    want, tol, _ = reference(y.double().numpy(), target[2:].numpy(), sup.numpy(), 3)
    near(o["lse"][2:], want["lse"], tol)
    assert np.array_equal(o["top_id"][2:].cpu().numpy(), want["top_id"])
    y = x[:1].clone()
    y[0, 5] = -float("inf")
    y[0, 7] = -float("inf")
    assert o["top_id"][0].cpu().tolist() == torch.sort(y[0], descending=True, stable=True).indices[:3].tolist()
    assert o["top_id"][1, 0].item() == 6


@pytest.mark.parametrize("outputs", [("logp",), ("entropy",), ("lse", "top_id"), ("top_logp",), ("top_id",)])
def test_outputs_left_out(cuda, outputs):
    gen = torch.Generator().manual_seed(9)
    x = torch.randn((3, 5000), generator=gen)
    target = torch.tensor([5, 6, 7], dtype=torch.int32)
    o = buffers(3, 4)
    P = lambda n: o[n].data_ptr() if n in outputs else None  # noqa: E731
    xd, td = x.cuda(), target.cuda()
    out = Logprobs(td.data_ptr() if "logp" in outputs else None, P("logp"), P("entropy"), P("lse"), P("top_id"),
                   P("top_logp"), 1, None, 4 if "top_id" in outputs or "top_logp" in outputs else 0)
    rc = m.lib.mmz_token_logprobs(xd.data_ptr(), 5000, 1, 3, 5000, None, ctypes.byref(out),
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    want, tol, etol = reference(x.double().numpy(), target.numpy(), None, 4)
    for n in o:
        if n not in outputs:
            assert (o[n] == 77).all()
        elif n == "top_id":
            assert np.array_equal(o[n].cpu().numpy(), want[n])
        else:
            near(o[n], want[n], (etol if n == "entropy" else tol)[:, None] * np.ones(4) * 2 if n == "top_logp" else
                 (etol if n == "entropy" else 2 * tol))


def test_columns_of_a_captured_step(cuda):
    """Target and outputs as [rows][steps], the column read from device memory: a captured call replayed along them; a
    counter outside the columns writes nothing."""
    gen = torch.Generator().manual_seed(10)
    rows, V, steps, top = 3, 3000, 5, 2
    x = torch.randn((steps, rows, V), generator=gen).half()
    target = torch.randint(0, V, (rows, steps), generator=gen, dtype=torch.int32)
    cur = torch.empty((rows, V), dtype=torch.float16, device="cuda")
    col = torch.zeros(1, dtype=torch.int32, device="cuda")
    td = target.cuda()
    o = dict(logp=torch.full((rows, steps), 77.0, device="cuda"), entropy=torch.full((rows, steps), 77.0, device="cuda"),
             lse=torch.full((rows, steps), 77.0, device="cuda"),
             top_id=torch.full((rows, steps, top), 77, dtype=torch.int32, device="cuda"),
             top_logp=torch.full((rows, steps, top), 77.0, device="cuda"))
    cur.zero_()
    st = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=st):
        m.token_logprobs(cur, td, **o, col=col)
    for t in list(range(steps - 1)) + [-1, steps]:
        if 0 <= t < steps:
            cur.copy_(x[t])
        col.fill_(t)
        g.replay()
    torch.cuda.synchronize()
    for t in range(steps - 1):
        ref = reference(x[t].double().numpy(), target[:, t].numpy(), None, top)
        compare({n: v[:, t] for n, v in o.items()}, ref, top)
    assert all((v[:, steps - 1] == 77).all() for v in o.values())


def test_refusals(cuda):
    x = torch.zeros((2, 10), dtype=torch.float16, device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.zeros(2, device="cuda")
    emb = torch.zeros((10, 64), dtype=torch.float16, device="cuda")
    h = torch.zeros((2, 64), dtype=torch.float16, device="cuda")
    t2, f2 = t[:, None].contiguous(), f[:, None].contiguous()
    bad = [lambda: m.token_logprobs(x.double(), t, f), lambda: m.token_logprobs(x, t.long(), f),
           lambda: m.token_logprobs(x, t, f.half()), lambda: m.token_logprobs(x, t[:1], f), lambda: m.token_logprobs(x.t(), t, f),
           lambda: m.token_logprobs(x, t, f, top_id=torch.zeros((2, 9), dtype=torch.int32, device="cuda")),
           lambda: m.token_logprobs(x, t, f, top_id=torch.zeros((2, 3), dtype=torch.int32, device="cuda"), top_logp=f2),
           lambda: m.token_logprobs(x, t, f, sup=torch.zeros(9, dtype=torch.uint8, device="cuda")),
           lambda: m.token_logprobs(x, t, f, col=t[:1]), lambda: m.token_logprobs(x, t2, f2, col=t[:0]),
           lambda: m.token_logprobs(x, None, f), lambda: m.token_logprobs(x[:, :0], t, f),
           lambda: m.linear_logprobs(h[:, :32], emb[:, :32].contiguous(), t, f), lambda: m.linear_logprobs(h, emb[:, :32], t, f),
           lambda: m.linear_logprobs(h.float(), emb, t, f), lambda: m.linear_logprobs(h, emb.cpu(), t, f),
           lambda: m.linear_logprobs(h, emb, t, f, scratch=torch.zeros(16, dtype=torch.uint8, device="cuda"))]
    for call in bad:
        with pytest.raises(m.MmzError):
            call()
    m.token_logprobs(x[:0], t[:0], f[:0])  # no rows: nothing to do
    m.linear_logprobs(h[:0], emb, t[:0], f[:0])


def test_row_offsets_past_32_bits(cuda):
    V, ld = 1000, (1 << 31) + 8
    big = torch.empty(ld + V, dtype=torch.float16, device="cuda")
    x = big.as_strided((2, V), (ld, 1))
    gen = torch.Generator().manual_seed(11)
    val = torch.randn((2, V), generator=gen).half()
    x.copy_(val)
    o = buffers(2, 5)
    target = torch.tensor([3, 999], dtype=torch.int32)
    m.token_logprobs(x, target.cuda(), **o)
    compare(o, reference(val.double().numpy(), target.numpy(), None, 5), 5)


def grid_states(gen, rows, V, d):
    """Hidden states and an embedding whose products' partial sums are exact in fp32: multiples of 2^-5 and 2^-10."""
    emb = (torch.randn((V, d), generator=gen) * (1.6 / d ** 0.5) * 1024).round() / 1024
    x = (torch.randn((rows, d), generator=gen) * 32).round() / 32
    return x.half(), emb.half()


HIDDEN = [(1, 1, 64, 1), (2, 5, 64, 8), (1, 51865, 384, 5), (3, 1000, 128, 5), (32, 3001, 1280, 8), (33, 2000, 192, 0),
          (31, 131, 64, 3), (64, 700, 64, 2), (100, 5000, 384, 5), (128, 257, 64, 8), (129, 1024, 256, 5),
          (257, 777, 64, 5), (1000, 2049, 128, 4), (300, 20000, 64, 5), (8, 60000, 64, 5), (513, 256, 1280, 5),
          (20000, 600, 64, 3), (3000, 3001, 64, 8), (130, 51866, 384, 5)]


@pytest.mark.parametrize("shape", HIDDEN)
@pytest.mark.parametrize("masked", [False, True])
def test_hidden_states(cuda, shape, masked):
    rows, V, d, top = shape
    gen = torch.Generator().manual_seed(rows + V)
    x, emb = grid_states(gen, rows, V, d)
    target = torch.randint(-1, V + 1, (rows,), generator=gen, dtype=torch.int32)
    sup = (torch.rand(V, generator=gen) < 0.3).to(torch.uint8) if masked else None
    wide = torch.empty((rows, d + 8), dtype=torch.float16, device="cuda")  # a row pitch wider than the states
    wide.fill_(float("nan"))
    xd = wide[:, :d]
    xd.copy_(x)
    o = buffers(rows, top)
    m.linear_logprobs(xd, emb.cuda(), target.cuda(), **o, sup=None if sup is None else sup.cuda())
    logits = (x.cuda().double() @ emb.cuda().double().t()).cpu().numpy()
    compare(o, reference(logits, target.numpy(), None if sup is None else sup.numpy(), top), top)
    assert m.status()[0] == 0


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape", [(1, 3001, 384, 5), (20, 5000, 1280, 8), (33, 2000, 192, 3), (100, 1000, 1280, 5),
                                   (130, 3000, 1280, 5), (300, 2500, 320, 8)])
def test_hidden_states_off_any_grid(cuda, shape, masked):
    """fp16 states and embeddings as they come, whose partial sums are not exact. A product takes 16 terms at a time: each
    of them, the sum so far and the new sum lose less than 2^-23 of the largest of these numbers (P, over the whole
    product, in 64 bits). So a logit is off by at most D = 18 d / 16 2^-23 P (its row's largest), lse and the k-th largest
    logit by D, a log probability by 2 D, and the entropy, whose derivatives -p (log p + H) sum to 2 H at most in
    magnitude, by 2 H D (a tenth more for its second order, D being below 0.01). The alternatives are those of logits that
    lie so close to the exact ones: their own logits come within 2 D of the k-th largest, and where no two of the
    largest top + 1 are that close, they are the same."""
    rows, V, d, top = shape
    gen = torch.Generator().manual_seed(rows + d)
    x = torch.randn((rows, d), generator=gen).half()
    emb = (torch.randn((V, d), generator=gen) * (1.6 / d ** 0.5)).half()
    target = torch.randint(0, V, (rows,), generator=gen, dtype=torch.int32)
    sup = (torch.rand(V, generator=gen) < 0.3).to(torch.uint8) if masked else None
    xd, ed = x.cuda(), emb.cuda()
    o = buffers(rows, top)
    m.linear_logprobs(xd, ed, target.cuda(), **o, sup=None if sup is None else sup.cuda())
    logits, D = np.empty((rows, V)), np.empty(rows)
    e64 = ed.double()
    for r in range(rows):
        terms = e64 * xd[r].double()
        sums = terms.view(V, d // 16, 16).sum(2).cumsum(1)
        logits[r] = sums[:, -1].cpu().numpy()
        D[r] = 18 * d / 16 * 2.0 ** -23 * max(terms.abs().max().item(), sums.abs().max().item())
    assert D.max() < 0.01
    want, tol, etol = reference(logits, target.numpy(), None if sup is None else sup.numpy(), top + 1)
    near(o["lse"], want["lse"], tol + D)
    fin = np.where(np.isinf(want["logp"]), 0, np.abs(want["logp"]))
    near(o["logp"], want["logp"], tol + fin * 2.0 ** -22 + 2 * D)
    near(o["entropy"], want["entropy"], etol + 2.2 * want["entropy"] * D)
    tlp = want["top_logp"]
    near(o["top_logp"], tlp[:, :top], (tol + 2 * D)[:, None] + np.abs(tlp[:, :top]) * 2.0 ** -22)
    ids = o["top_id"].cpu().numpy()
    if sup is not None:
        logits[:, sup.numpy() != 0] = -np.inf
    clear = 0
    for r in range(rows):
        assert len(set(ids[r])) == top
        kth = tlp[r, :top] + want["lse"][r]
        assert (np.abs(logits[r, ids[r]] - kth) <= 2 * D[r] + 1e-12).all()
        if (-np.diff(tlp[r]) > 2 * D[r]).all():
            assert np.array_equal(ids[r], want["top_id"][r, :top])
            clear += 1
    assert clear > 0.8 * rows
    assert m.status()[0] == 0


def test_hidden_states_ties_and_rows_that_repeat(cuda):
    """Equal embedding rows tie (the lower id first), equal hidden states give equal rows, a zero state a uniform one."""
    gen = torch.Generator().manual_seed(12)
    x, emb = grid_states(gen, 40, 1500, 128)
    emb[700:] = emb[:800].clone()
    x[7] = x[33]
    x[9] = 0
    o = buffers(40, 8)
    target = torch.randint(0, 1500, (40,), generator=gen, dtype=torch.int32)
    target[7] = target[33]
    m.linear_logprobs(x.cuda(), emb.cuda(), target.cuda(), **o)
    logits = x.double().numpy() @ emb.double().numpy().T
    compare(o, reference(logits, target.numpy(), None, 8), 8)
    for v in o.values():
        assert torch.equal(v[7], v[33])


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_hidden_states_with_nan(cuda, rows):
    """A NaN in an id's embedding makes every row's sums NaN and is no alternative; in a hidden state, that row's alone;
    suppressed, it is not read into anything."""
    gen = torch.Generator().manual_seed(15)
    x, emb = grid_states(gen, rows, 700, 64)
    emb[33, 5] = float("nan")
    target = torch.full((rows,), 3, dtype=torch.int32)
    logits = x.double().numpy() @ np.nan_to_num(emb.double().numpy()).T
    logits[:, 33] = -np.inf
    sup = torch.zeros(700, dtype=torch.uint8)
    for top in (1, 5):
        o = buffers(rows, top)
        m.linear_logprobs(x.cuda(), emb.cuda(), target.cuda(), **o, sup=sup.cuda())
        assert torch.isnan(torch.cat([o["lse"], o["logp"], o["entropy"]])).all()
        assert np.array_equal(o["top_id"].cpu().numpy(), reference(logits, target.numpy(), None, top)[0]["top_id"])
        sup[33] = 1
        o = buffers(rows, top)
        m.linear_logprobs(x.cuda(), emb.cuda(), target.cuda(), **o, sup=sup.cuda())
        compare(o, reference(logits, target.numpy(), None, top), top)
        sup[33] = 0
    emb[33, 5] = 0
    x[1, 7] = float("nan")
    o = buffers(rows, 5)
    m.linear_logprobs(x.cuda(), emb.cuda(), target.cuda(), **o)
    x[1] = 0
    want, tol, _ = reference(x.double().numpy() @ emb.double().numpy().T, target.numpy(), None, 5)
    ok = torch.arange(rows) != 1
    assert torch.isnan(o["lse"][1]) and (o["top_id"][1] == -1).all()
    near(o["lse"][ok.cuda()], want["lse"][ok.numpy()], tol[ok.numpy()])
    assert np.array_equal(o["top_id"].cpu().numpy()[ok.numpy()], want["top_id"][ok.numpy()])


def test_hidden_states_beside_the_greedy_choice(cuda):
    """The engine's logits_argmax and the first alternative agree where the best two logits are a step of fp16 apart."""
    gen = torch.Generator().manual_seed(13)
    rows, V, d = 16, 51866, 1280
    x, emb = grid_states(gen, rows, V, d)
    xd, ed = x.cuda(), emb.cuda()
    sup = torch.zeros(V, dtype=torch.uint8, device="cuda")
    tok = torch.zeros((rows, 8), dtype=torch.int32, device="cuda")
    done = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ctr = torch.zeros(4, dtype=torch.int32, device="cuda")
    ctr[0] = 3
    scratch = torch.zeros(m.logits_argmax_scratch_bytes(), dtype=torch.uint8, device="cuda")
    m.logits_argmax(xd, ed, sup, tok, done, ctr, 8, 1, 50257, scratch=scratch)
    o = buffers(rows, 2)
    m.linear_logprobs(xd, ed, tok[:, 4].contiguous(), **o, sup=sup)
    torch.cuda.synchronize()
    first, gap = o["top_id"][:, 0], (o["top_logp"][:, 0] - o["top_logp"][:, 1]).cpu().numpy()
    best = (o["top_logp"][:, 0] + o["lse"]).abs().cpu().numpy()
    clear = gap > 2 * best * 2.0 ** -10
    assert clear.sum() >= 4
    assert (first == tok[:, 4]).cpu().numpy()[clear].all()
    assert torch.allclose(o["logp"].cpu()[clear], o["top_logp"][:, 0].cpu()[clear])


def test_scoring_on_another_stream(cuda):
    gen = torch.Generator().manual_seed(14)
    x, emb = grid_states(gen, 50, 3000, 256)
    xd, ed, target = x.cuda(), emb.cuda(), torch.arange(50, dtype=torch.int32, device="cuda")
    a, b = buffers(50, 5), buffers(50, 5)
    m.linear_logprobs(xd, ed, target, **a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    scratch = torch.empty(m.linear_logprobs_scratch_bytes(50, 3000, 256), dtype=torch.uint8, device="cuda")
    m.linear_logprobs(xd, ed, target, **b, scratch=scratch, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_scratch_is_no_memory_of_the_current_stream(cuda):
    """As in the attention's test: a freed tensor that the current stream has yet to read, and calls without scratch on
    both streams in turn."""
    gen = torch.Generator().manual_seed(16)
    states = [grid_states(gen, 50, 3000, 256) for _ in "ab"]
    states = [(x.cuda(), emb.cuda()) for x, emb in states]
    target = torch.arange(50, dtype=torch.int32, device="cuda")
    want = [buffers(50, 5) for _ in "ab"]
    for (x, emb), o in zip(states, want):
        m.linear_logprobs(x, emb, target, **o)
    st = torch.cuda.Stream()
    outs = [buffers(50, 5) for _ in range(41)]
    held = torch.full((m.linear_logprobs_scratch_bytes(50, 3000, 256),), 7, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    torch.cuda._sleep(100000000)
    read = held.clone()
    del held
    m.linear_logprobs(*states[0], target, **outs[40], stream=st)
    for i in range(0, 40, 2):
        m.linear_logprobs(*states[0], target, **outs[i])
        m.linear_logprobs(*states[1], target, **outs[i + 1], stream=st)
    torch.cuda.synchronize()
    assert (read == 7).all()
    assert all(torch.equal(o[n], want[i & 1][n]) for i, o in enumerate(outs) for n in o)
