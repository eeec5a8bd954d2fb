"""The engine on the 8-bit cross k/v and with log probabilities: against its own fp16 cache, and the steps' logits."""
import ctypes

import numpy as np
import pytest
import torch

import mimizuku_b200 as m

pytestmark = pytest.mark.gpu


class Dev:
    def __init__(self, ptr, shape, typestr):
        self.__cuda_array_interface__ = {"shape": shape, "typestr": typestr, "data": (ptr, False), "version": 2}


def view(e, name, shape, typestr="<f2"):
    return torch.as_tensor(Dev(e.buffer(name), shape, typestr), device="cuda")


def clips(n, seed=0):
    ys = [m.synth_clip(seed + i, 160000 + 16000 * i) for i in range(n)]
    return m.log_mel_batch(ys, m.TINY.n_mels)


def engine(b, **kw):
    return m.Engine(m.TINY, bmax=b, eg=min(b, 4), seed=3, suppress=[1, 2, 7, 220], **kw)


@pytest.mark.parametrize("b", [1, 3, 12, 32])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_cross_attention_of_a_step(cuda, b, kind):
    """One decoding step on the 8-bit cache against the same on fp16. The last layer's attention output and the recorded
    probabilities move by what rounding moves them: an int8 code is off by at most half a step, of a scale of at most
    the 64 x 64 block's maximum / 127 (about 4.5 standard deviations: rms 1.0 % of a standard deviation), an e4m3 one by
    2^-4 of its value at most (rms below 2.7 %); the mean over 1500 positions shrinks error and output alike, and the
    keys' part (through scores far below 1) is no larger than the values': below 3 % and 8 % of the output's norm."""
    cfg, na = m.TINY, m.TINY.n_align
    mel, frames = clips(b)
    e = engine(b)
    h = torch.from_numpy(mel).cuda().half()
    for g in range(0, b, 4):
        e.encode(h[g:g + 4].contiguous(), min(4, b - g), g)
    got = {}
    for k in ("fp16", kind):
        e.xkv = k
        assert e.xkv == k
        e.reset(np.tile(np.array([cfg.prompt], np.int32), (b, 1)))
        view(e, "align", (b, cfg.max_t, na, 1500)).zero_()
        e.step(b, len(cfg.prompt))
        e.sync()
        got[k] = (view(e, "att", (b, cfg.d)).float().cpu().numpy(),
                  view(e, "align", (b, cfg.max_t, na, 1500)).float().cpu().numpy())
    lim = 0.03 if kind == "int8" else 0.08
    (o16, a16), (o8, a8) = got["fp16"], got[kind]
    assert np.isfinite(o8).all()
    assert 0 < np.linalg.norm(o8 - o16) < lim * np.linalg.norm(o16)
    assert np.allclose(a8[:, 0].sum(-1), 1, atol=2e-3) and not a8[:, 1:].any()
    assert np.linalg.norm(a8 - a16) < lim * np.linalg.norm(a16)
    assert m.status()[0] == 0
    e.close()


def test_back_to_fp16_gives_the_same_as_ever(cuda):
    mel, frames = clips(2)
    e = engine(2)
    a = e.transcribe(mel, frames, max_new=12)
    e.xkv = "int8"
    r8 = e.transcribe(mel, frames, max_new=12)
    assert (r8["lens"] >= len(m.TINY.prompt)).all() and (r8["tokens"] < m.TINY.vocab).all()
    again = e.transcribe(mel, frames, max_new=12)
    e.xkv = "fp16"
    b = e.transcribe(mel, frames, max_new=12)
    for k in ("tokens", "lens", "times"):
        assert np.array_equal(a[k], b[k]) and np.array_equal(r8[k], again[k]), k
    e.close()


@pytest.mark.parametrize("b,kind", [(2, "fp16"), (2, "int8"), (12, "fp16"), (32, "int8")])
def test_logprobs_of_a_transcription(cuda, b, kind):
    """The log probabilities and entropies against 64 bits of each step's own logits, and unchanged tokens."""
    cfg, new = m.TINY, 10
    mel, frames = clips(b)
    e = engine(b)
    e.xkv = kind
    plain = e.transcribe(mel, frames, max_new=new)
    assert "logprobs" not in plain
    e.logprobs = True
    r = e.transcribe(mel, frames, max_new=new)
    for k in ("tokens", "lens", "times"):
        assert np.array_equal(plain[k], r[k]), k
    # the same steps one by one, the logits read after each
    np_ = len(cfg.prompt)
    e.reset(np.tile(np.array([cfg.prompt], np.int32), (b, 1)))
    want = np.zeros((b, cfg.max_t))
    ent = np.zeros((b, cfg.max_t))
    for p in range(np_ - 1 + new):
        e.step(b, np_)
        e.sync()
        if p + 1 < np_:
            continue
        x = view(e, "logits", (b, cfg.vocab)).double().cpu()
        x[:, [1, 2, 7, 220]] = -float("inf")
        lp = torch.log_softmax(x, 1)
        tok = torch.from_numpy(r["tokens"][:, p + 1].astype(np.int64))
        want[:, p + 1] = lp.gather(1, tok[:, None])[:, 0]
        ent[:, p + 1] = torch.special.entr(lp.exp()).sum(1)
    for s in range(b):
        lo, hi = np_, r["lens"][s]
        assert (r["logprobs"][s, :lo] == 0).all() and (r["logprobs"][s, hi:] == 0).all()
        assert (r["entropy"][s, :lo] == 0).all() and (r["entropy"][s, hi:] == 0).all()
        # fp32 sums of 51865 terms (as token_logprobs' tests derive it): below 1e-4
        assert np.abs(r["logprobs"][s, lo:hi] - want[s, lo:hi]).max() < 1e-4
        assert np.abs(r["entropy"][s, lo:hi] - ent[s, lo:hi]).max() < 1e-3
    e.logprobs = False
    assert "logprobs" not in e.transcribe(mel, frames, max_new=2)
    with pytest.raises(m.MmzError, match="set_logprobs"):
        m.engine._check(m.lib.mmz_engine_read_logprobs(e._h, None, None), "read_logprobs")
    e.close()


@pytest.mark.parametrize("b,graph", [(2, True), (12, True), (3, False)])
def test_the_first_token_is_chosen_without_the_begin_suppressed(cuda, b, graph):
    """Both ids that clip 0 would begin with are begin-suppressed: its first token's distribution is without them (and
    every clip's), the second token's with them. Random weights' logits are nearly equal, so that only 160 ids are left to
    choose from: two of them weigh some 2 / 160."""
    cfg, new = m.TINY, 3
    np_ = len(cfg.prompt)
    sup = [i for i in range(cfg.vocab) if i % 324]
    mel, frames = clips(b)
    prompts = np.tile(np.array([cfg.prompt], np.int32), (b, 1))

    def steps(e, n):
        """The logits that each of the n generated tokens is chosen from, in 64 bits."""
        e.reset(prompts)
        out = []
        for p in range(np_ - 1 + n):
            e.step(b, np_)
            e.sync()
            if p + 1 >= np_:
                out.append(view(e, "logits", (b, cfg.vocab)).double().cpu())
                out[-1][:, sup] = -float("inf")
        return out

    make = lambda **kw: m.Engine(cfg, bmax=b, eg=min(b, 4), seed=3, suppress=sup, **kw)  # noqa: E731
    e = make()
    e.transcribe(mel, frames, max_new=1)  # the clips are encoded
    ids = steps(e, 1)[0][0].topk(2).indices.tolist()
    e.close()
    e = make(begin_suppress=tuple(ids))
    e.logprobs = True
    r = e.transcribe(mel, frames, max_new=new, graph=graph)
    x = steps(e, new)
    left = torch.logsumexp(x[0], 1)
    x[0][:, ids] = -float("inf")
    # what the two weigh shows: 30 times the tolerance below
    assert (left - torch.logsumexp(x[0], 1))[0] > 3e-3
    for j in range(new):
        at = np_ + j
        lp = torch.log_softmax(x[j], 1)
        want = lp.gather(1, torch.from_numpy(r["tokens"][:, at].astype(np.int64))[:, None])[:, 0]
        ent = torch.special.entr(lp.exp()).sum(1)
        live = torch.from_numpy(r["lens"].astype(np.int64)) > at
        assert j or (live.all() and not np.isin(r["tokens"][:, at], ids).any())
        # (as in the test above)
        assert (torch.from_numpy(r["logprobs"][:, at]).double() - want)[live].abs().max() < 1e-4
        assert (torch.from_numpy(r["entropy"][:, at]).double() - ent)[live].abs().max() < 1e-3
    e.close()


def test_finished_sequences_are_left_out(cuda):
    """A finished sequence's attention output is zero and its recorded probabilities stay as they were."""
    cfg, b = m.TINY, 12
    mel, frames = clips(b)
    e = engine(b)
    h = torch.from_numpy(mel).cuda().half()
    for g in range(0, b, 4):
        e.encode(h[g:g + 4].contiguous(), min(4, b - g), g)
    e.xkv = "int8"
    e.reset(np.tile(np.array([cfg.prompt], np.int32), (b, 1)))
    align = view(e, "align", (b, cfg.max_t, cfg.n_align, 1500))
    align.fill_(5)
    done = view(e, "done", (b,), "<i4")
    done[::3] = 1
    torch.cuda.synchronize()
    e.step(b, len(cfg.prompt))
    e.sync()
    att = view(e, "att", (b, cfg.d))
    fin = torch.arange(b, device="cuda") % 3 == 0
    assert (att[fin] == 0).all() and (att[~fin] != 0).any(1).all()
    assert (align[fin] == 5).all() and (align[~fin][:, 0] <= 1).all() and (align[:, 1:] == 5).all()
    e.close()


def test_settings_refuse(cuda):
    e = engine(1)
    for call in (lambda: m.lib.mmz_engine_set_xkv(e._h, 3), lambda: m.lib.mmz_engine_set_xkv(None, 1),
                 lambda: m.lib.mmz_engine_set_logprobs(e._h, 2), lambda: m.lib.mmz_engine_read_logprobs(e._h, None, None),
                 lambda: m.lib.mmz_engine_set_logprobs(None, 1)):
        assert call() != 0 and m.lib.mmz_last_error()
    with pytest.raises(m.MmzError):
        e.xkv = "int4"
    assert e.xkv == "fp16" and not e.logprobs
    e.close()


def test_logprobs_are_those_of_a_transcription_since_the_setting(cuda):
    mel, frames = clips(1)
    e = engine(1)
    read = lambda: m.lib.mmz_engine_read_logprobs(e._h, None, None)
    e.transcribe(mel, frames, max_new=2)
    e.logprobs = True  # after the transcription, which left none
    assert read() == -1 and b"a transcription come first" in m.lib.mmz_last_error()
    e.transcribe(mel, frames, max_new=2)
    assert read() == 0
    e.reset(np.array([m.TINY.prompt], np.int32))  # the next steps write over them
    assert read() == -1
    e.logprobs = False
    e.logprobs = True
    assert read() == -1
    e.close()
