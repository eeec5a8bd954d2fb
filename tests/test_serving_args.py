"""The 8-bit cache and the log probabilities refuse bad arguments on the host, before a device is touched."""
import ctypes

import pytest

import mimizuku_b200 as m

L = m.lib
A = 1 << 20  # an aligned address that nothing reads


class Kv8(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [
        (n, ctypes.c_longlong) for n in ("seq", "head", "scale_seq", "scale_head")] + [
        (n, ctypes.c_int) for n in ("heads", "cap", "block", "kind")]


class Attn8(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("qs", ctypes.c_longlong * 3), ("out", ctypes.c_void_p),
                ("os", ctypes.c_longlong * 3)] + [(n, ctypes.c_void_p) for n in ("lens", "probs", "pslot", "scratch")] + [
        ("scratch_bytes", ctypes.c_ulonglong)] + [(n, ctypes.c_int) for n in ("batch", "rows", "q_heads", "slots", "causal")] + [
        ("scale", ctypes.c_float)]


class Logprobs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("target", "logp", "entropy", "lse", "top_id", "top_logp")] + [
        ("ld", ctypes.c_longlong), ("col", ctypes.c_void_p), ("top", ctypes.c_int)]


def cache(k8=A, v8=A, ks=A, vs=A, cs=(6400, 6400), heads=1, cap=100, block=64, kind=0):
    return Kv8(k8, v8, ks, vs, *cs, 2, 2, heads, cap, block, kind)


def write(k=A, v=A, xs=(64, 64, 64), batch=1, n=1, **kw):
    return L.mmz_kv8_write(ctypes.byref(cache(**kw)), k, v, *xs, None, batch, n, None)


def read(k=A, v=A, xs=(64, 64, 64), batch=1, n=1, **kw):
    return L.mmz_kv8_read(ctypes.byref(cache(**kw)), k, v, *xs, None, None, batch, n, None)


def test_null_structs_are_refused():
    for call in (lambda: L.mmz_kv8_write(None, A, A, 64, 64, 64, None, 1, 1, None), lambda: L.mmz_attn8(None, None, None),
                 lambda: L.mmz_kv8_read(None, A, A, 64, 64, 64, None, None, 1, 1, None),
                 lambda: L.mmz_token_logprobs(A, 9, 0, 1, 9, None, None, None),
                 lambda: L.mmz_linear_logprobs(A, 64, A, 1, 9, 64, None, None, None, 0, None)):
        assert call() == -1 and b"null" in L.mmz_last_error()


@pytest.mark.parametrize("fn,name", [(write, b"kv8_write"), (read, b"kv8_read")])
@pytest.mark.parametrize("bad,word", [
    (dict(block=0), b"block"), (dict(block=48), b"block"), (dict(block=256), b"block"), (dict(kind=2), b"kind"),
    (dict(kind=-1), b"kind"), (dict(batch=-1), b"batch"), (dict(heads=0), b"heads"), (dict(n=-1), b"n >= 0"),
    (dict(cap=0), b"cap"), (dict(cap=0x7fffffff), b"cap"), (dict(k=None), b"null"), (dict(ks=None), b"null"), (dict(v8=None), b"null"),
    (dict(k=A + 8), b"aligned"), (dict(k8=A + 4), b"aligned"), (dict(xs=(64, 60, 64)), b"strides"),
    (dict(cs=(6400, 6392)), b"strides"),
    (dict(batch=1 << 20, heads=1 << 12, n=99, cs=(1 << 40, 6400)), b"2^31")])
def test_cache_calls_refuse(fn, name, bad, word):
    assert fn(**bad) == -1
    msg = L.mmz_last_error()
    assert name in msg and word in msg


def test_a_cache_that_overlaps_is_read_only():
    for bad in (dict(batch=2, cs=(0, 6400)), dict(heads=2, cs=(12800, 3200)), dict(batch=2, cs=(6384, 6400))):
        assert write(**bad) == -1 and b"overlap" in L.mmz_last_error()


def test_sequences_that_start_where_heads_do_overlap():
    # each stride alone is wide enough: sequence 1's first head lies on sequence 0's second
    assert write(batch=2, heads=2, cs=(6400, 6400)) == -1 and b"overlap" in L.mmz_last_error()
    assert write(batch=2, heads=2, cs=(12800, 6400)) == -1 and b"overlap" in L.mmz_last_error()  # (the scales: 2 and 2)


def test_outputs_in_one_place_are_refused():
    for xs in ((0, 64, 64), (64, 128, 128), (4096, 64, 64), (1024, 64, 120)):
        assert read(batch=2, n=2, heads=2, xs=xs) == -1 and b"overlap" in L.mmz_last_error()
        assert attend(batch=2, rows=2, hq=2, hkv=2, os=xs) == -1 and b"overlap" in L.mmz_last_error()
    for xs in ((256, 128, 64), (64, 256, 128), (-256, 64, 128), (1 << 62, 128, 64)):  # any order that nests is one
        assert attend(batch=2, rows=2, hq=2, hkv=2, os=xs, probs=A, pslot=A, slots=1) == -1
        assert b"scratch" in L.mmz_last_error()  # the next check


def test_keys_and_values_in_one_place_are_refused():
    far = 1 << 30
    # one cache for both, the values a position further on, one sequence's values on the next one's keys; the scales alike
    for bad in (dict(), dict(v8=A + 64), dict(batch=2, cs=(12800, 6400), v8=A + 12800), dict(v8=A - 6336),
                dict(v8=A + far), dict(v8=A + far, vs=A + 4), dict(v8=A + far, batch=2, cs=(12800, 6400), vs=A - 8)):
        assert write(**bad) == -1 and b"kv8_write: the cache's keys and values overlap" in L.mmz_last_error()
    for bad in (dict(), dict(v=A + 16), dict(v=A + 112, n=3), dict(v=A - 256, n=3, xs=(64, 128, 64)),
                dict(v=A + 256, n=2, heads=2, xs=(64, 128, 64))):
        assert read(**bad) == -1 and b"kv8_read: k and v overlap" in L.mmz_last_error()


def test_an_output_over_other_rows_of_q_is_refused():
    dims = dict(batch=2, rows=3, hq=2, hkv=2)
    for bad in (dict(out=A + 16), dict(out=A - 112), dict(dims, qs=(384, 128, 64), os=(384, 128, 64), out=A + 128),
                dict(dims, qs=(384, 128, 64), os=(384, 64, 192)),  # the same rows in another order
                dict(dims, qs=(1152, 384, 64), os=(1152, 384, 64), out=A + 768),
                dict(dims, qs=(0, 128, 64), os=(384, 128, 64), out=A + 640),
                dict(dims, qs=(384, 128, 64), os=(-384, 128, 64), out=A + 1536)):
        assert attend(**bad) == -1 and b"attn8: out over q, and not q itself" in L.mmz_last_error()


def test_nothing_to_do_is_no_error():
    assert write(batch=0, k=None) == 0 and write(n=0, k=None) == 0
    assert read(batch=0) == 0 and read(n=0) == 0
    assert attend(batch=0, q=None) == 0 and attend(rows=0) == 0
    assert logits(rows=0, x=None) == 0 and hidden(rows=0, x=None) == 0


def attend(q=A, qs=(64, 64, 64), out=A, os=(64, 64, 64), batch=1, rows=1, hq=1, hkv=1, probs=None, pslot=None, slots=0,
           scratch=None, sb=0, **kw):
    a = Attn8(q, (ctypes.c_longlong * 3)(*qs), out, (ctypes.c_longlong * 3)(*os), None, probs, pslot, scratch, sb, batch, rows,
              hq, slots, 0, 0.125)
    return L.mmz_attn8(ctypes.byref(cache(heads=hkv, **kw)), ctypes.byref(a), None)


@pytest.mark.parametrize("bad,word", [
    (dict(block=8), b"block"), (dict(kind=3), b"kind"), (dict(hq=3, hkv=2), b"multiple of kv_heads"),
    (dict(hkv=0), b"heads"), (dict(batch=-1), b"batch"), (dict(rows=-1), b"rows"), (dict(cap=0), b"cap"),
    (dict(slots=-1), b"cap"), (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(ks=None), b"null"),
    (dict(probs=A), b"pslot"), (dict(q=A + 2), b"aligned"), (dict(out=A + 8), b"aligned"),
    (dict(probs=A + 8, pslot=A, slots=1), b"aligned"), (dict(qs=(64, 64, 63)), b"strides"),
    (dict(os=(64, 4, 64)), b"strides"), (dict(cs=(6401, 6400)), b"strides"), (dict(cap=0x7fffffff), b"cap"),
    (dict(probs=A, pslot=A, slots=1), b"scratch"), (dict(probs=A, pslot=A, slots=1, scratch=A + 8, sb=1 << 20), b"scratch"),
    (dict(probs=A, pslot=A, slots=1, scratch=A, sb=4), b"scratch"), (dict(cap=100000), b"scratch"),
    (dict(batch=1 << 20, hq=1 << 12, hkv=1 << 12), b"2^31"), (dict(rows=0x7fffffff), b"rows")])
def test_attention_refuses(bad, word):
    assert attend(**bad) == -1
    msg = L.mmz_last_error()
    assert b"attn8" in msg and word in msg


def outs(target=A, logp=A, top=0, ld=1):
    return ctypes.byref(Logprobs(target, logp, None, None, None, None, ld, None, top))


def logits(x=A, ldx=100, type=0, rows=1, vocab=100, **kw):
    return L.mmz_token_logprobs(x, ldx, type, rows, vocab, None, outs(**kw), None)


def hidden(x=A, ldx=64, emb=A, rows=1, vocab=100, d=64, scratch=None, sb=0, **kw):
    return L.mmz_linear_logprobs(x, ldx, emb, rows, vocab, d, None, outs(**kw), scratch, sb, None)


@pytest.mark.parametrize("bad,word", [
    (dict(type=2), b"type"), (dict(rows=-1), b"rows"), (dict(vocab=0), b"vocab"), (dict(ldx=99), b"ldx"),
    (dict(top=9), b"alternatives"), (dict(top=-1), b"alternatives"), (dict(ld=0), b"stride"),
    (dict(target=None), b"target"), (dict(x=None), b"null"), (dict(x=A + 1), b"aligned"),
    (dict(x=A + 2, type=1), b"aligned")])
def test_token_logprobs_refuses(bad, word):
    assert logits(**bad) == -1
    msg = L.mmz_last_error()
    assert b"token_logprobs" in msg and word in msg


@pytest.mark.parametrize("bad", [dict(rows=0x7fffffff), dict(rows=0x7ffffc01), dict(rows=0x7fffffff, type=1),
                                 dict(vocab=0x7fffffff, ldx=0x7fffffff), dict(rows=0x7fffffff, x=None)])
def test_rows_and_ids_near_2_to_31_are_refused(bad):
    assert logits(**(dict(vocab=1, ldx=1) | bad)) == -1
    assert b"token_logprobs: vocab up to 2^31 - 16, rows up to 2^31 - 1024" in L.mmz_last_error()


@pytest.mark.parametrize("bad,word", [
    (dict(d=96), b"width"), (dict(d=0), b"width"), (dict(rows=-1), b"rows"), (dict(vocab=0), b"vocab"),
    (dict(top=9), b"alternatives"), (dict(ld=0), b"stride"), (dict(target=None), b"target"), (dict(x=None), b"aligned"),
    (dict(emb=A + 8), b"aligned"), (dict(ldx=56), b"ldx"), (dict(ldx=68), b"pitch"), (dict(scratch=None), b"scratch"),
    (dict(scratch=A, sb=1), b"scratch"), (dict(scratch=A + 8, sb=1 << 30), b"scratch")])
def test_linear_logprobs_refuses(bad, word):
    assert hidden(**bad) == -1
    msg = L.mmz_last_error()
    assert b"linear_logprobs" in msg and word in msg


def test_scratch_sizes():
    assert L.mmz_attn8_scratch_bytes(0, 1, 1, 1, 1, 0) == 0 and L.mmz_attn8_scratch_bytes(1, 1, 1, 2, 1, 0) == 0
    assert L.mmz_linear_logprobs_scratch_bytes(0, 1, 64) == 0 and L.mmz_linear_logprobs_scratch_bytes(1, 1, 0) == 0
    assert m.linear_logprobs_scratch_bytes(7, 51866, 1280) % 16 == 0


def test_sizes_whose_products_pass_64_bits():
    big, top = 1 << 30, 0x7fffffff
    for rows, vocab in ((top, top), (top, 1), (1, top), (top, 1 << 30), (0x7fffff01, 0x40000000)):
        assert L.mmz_linear_logprobs_scratch_bytes(rows, vocab, 64) > 0
    for dims in ((big, top, big, big, top, 0), (big, top, big, 1, 1, 0), (top, top, 1, 1, top, top), (1 << 16, 1, 1, 1, 1 << 24, 1 << 24)):
        assert L.mmz_attn8_scratch_bytes(*dims) == 0
    wide = 1 << 40
    for bad in (dict(batch=big, heads=big, n=16), dict(batch=big, heads=1 << 31 >> 1, n=64)):
        for call in (write, read):
            assert call(cs=(wide, 6400), **bad) == -1 and b"2^31" in L.mmz_last_error()
    for bad in (dict(batch=big, rows=0x7fffff00, hq=big, hkv=big), dict(batch=big, hq=big, hkv=1),
                dict(batch=1 << 16, slots=1 << 24, cap=1 << 24, probs=A, pslot=A, scratch=A, sb=1 << 30)):
        assert attend(**bad) == -1 and b"attn8: too many rows" in L.mmz_last_error()


def test_python_calls_refuse_what_is_no_cuda_tensor():
    import torch
    k8 = torch.zeros((1, 2, 8, 64), dtype=torch.int8)
    s = torch.zeros((1, 2, 1))
    x = torch.zeros((1, 1, 2, 64), dtype=torch.float16)
    with pytest.raises(m.MmzError, match="not a CUDA tensor"):
        m.kv8_write(x, x, k8, k8, s, s)
    with pytest.raises(m.MmzError, match="not a CUDA tensor"):
        m.attn8(x, None, x, s, s, x)
    with pytest.raises(m.MmzError, match="not a CUDA tensor"):
        m.kv8_read(k8, k8, s, s, x, x, block=20)
    with pytest.raises(m.MmzError, match="fp16 or fp32"):
        m.token_logprobs(k8[0, 0], s, s)
    with pytest.raises(m.MmzError, match="are tensors"):
        m.linear_logprobs(None, x, s, s)
    with pytest.raises(m.MmzError, match="not a CUDA tensor"):
        m.linear_logprobs(x[0, 0], x[0, 0], s[0, 0], s[0, 0])
    with pytest.raises(AttributeError):
        m.no_such_call


def test_python_calls_take_their_arguments_by_name():
    import inspect
    for f, first, last in ((m.kv8_write, "k", "stream"), (m.kv8_read, "k8", "stream"), (m.attn8, "q", "stream"),
                           (m.token_logprobs, "logits", "stream"), (m.linear_logprobs, "x", "stream")):
        names = list(inspect.signature(f).parameters)
        assert (names[0], names[-1]) == (first, last) and f.__doc__
        with pytest.raises(TypeError, match="missing required argument"):
            f()
        with pytest.raises(TypeError, match="unexpected keyword argument 'colour'"):
            f(*[None] * 3, colour=1)
        with pytest.raises(TypeError, match="multiple values for argument"):
            f(None, **{first: None})
        with pytest.raises(TypeError, match="at most"):
            f(*[None] * (len(names) + 1))
        required = [n for n, p in inspect.signature(f).parameters.items() if p.default is p.empty]
        with pytest.raises(m.MmzError):
            f(**{"".join(n): None for n in names})  # every name is one, interned or not
        with pytest.raises(TypeError, match="missing required argument '%s'" % required[-1]):
            f(*[None] * (len(required) - 1))
