"""The 8-bit key/value cache (write, read back, attention) and the token log probabilities, over torch CUDA tensors.

Every call works on the current device and stream (or `stream`), checks its tensors on the host (MmzError) and returns
without waiting; outputs are tensors that the caller gives."""
import functools

import torch

from . import MmzError, _check, lib

_KIND = {torch.int8: 0, torch.float8_e4m3fn: 1}
_I32, _F16, _F32, _U8 = torch.int32, torch.float16, torch.float32, torch.uint8
_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _device(what, name, t):
    """The current device, which has to be tensor t's."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise MmzError(f"{what}: {name} is not a CUDA tensor")
    dev = t.get_device()
    if dev != _current():
        raise MmzError(f"{what}: {name} is on {t.device}, the current device is cuda:{_current()}")
    return dev


def _stream(stream, dev):
    if stream is None:
        return _raw_stream(dev)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _refuse(what, name, t, dtype, shape, dev):
    """Says what is wrong with a tensor that is no CUDA tensor of that dtype, shape (None: any) and device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise MmzError(f"{what}: {name} is not a CUDA tensor")
    if t.dtype is not dtype:
        raise MmzError(f"{what}: {name} is {t.dtype}, not {dtype}")
    if t.get_device() != dev:
        raise MmzError(f"{what}: {name} is on {t.device}, the current device is cuda:{dev}")
    if shape is not None and t.shape != shape:
        raise MmzError(f"{what}: {name} is {tuple(t.shape)}, not {tuple(shape)}")
    raise MmzError(f"{what}: {name} is not contiguous")


def _strided(what, name, t, dtype, shape, dev):
    """The address of a CUDA tensor of the current device with that dtype and shape."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != dev or t.shape != shape:
        _refuse(what, name, t, dtype, shape, dev)
    return t.data_ptr()


def _dense(what, name, t, dtype, shape, dev):
    """The same of a contiguous one; None for None."""
    if t is None:
        return None
    if (not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.get_device() != dev
            or shape is not None and t.shape != shape or not t.is_contiguous()):
        _refuse(what, name, t, dtype, shape, dev)
    return t.data_ptr()


def _cache(what, k8, v8, ks, vs, block, dev):
    """(batch, heads, cap, kind, pointers and strides) of a cache."""
    kind, shape = _KIND.get(k8.dtype), k8.shape
    if kind is None or len(shape) != 4 or shape[3] != 64:
        raise MmzError(f"{what}: k8 is an int8 or float8_e4m3fn tensor [batch][heads][cap][64]")
    if block not in (16, 32, 64, 128):
        raise MmzError(f"{what}: block is 16, 32, 64 or 128")
    b, h, cap, _ = shape
    blocks = (b, h, (cap + block - 1) // block)
    if not (isinstance(v8, torch.Tensor) and v8.dtype is k8.dtype and v8.shape == shape and v8.get_device() == dev):
        _refuse(what, "v8", v8, k8.dtype, shape, dev)
    for t, name in ((ks, "ks"), (vs, "vs")):
        if not (isinstance(t, torch.Tensor) and t.dtype is _F32 and t.shape == blocks and t.get_device() == dev):
            _refuse(what, name, t, _F32, blocks, dev)
    cs, ss = k8.stride(), ks.stride()
    if v8.stride() != cs or vs.stride() != ss:
        raise MmzError(f"{what}: keys and values of the cache have the same strides")
    if cs[3] != 1 or cap > 1 and cs[2] != 64 or blocks[2] > 1 and ss[2] != 1:
        raise MmzError(f"{what}: a head's rows of the cache, and its scales, lie one after another")
    # (the stride of a dimension of one may be anything)
    return b, h, cap, kind, (k8.data_ptr(), v8.data_ptr(), ks.data_ptr(), vs.data_ptr(), cs[0] if b > 1 else 0,
                             cs[1] if h > 1 else 0, ss[0] if b > 1 else 0, ss[1] if h > 1 else 0)


def _pair(what, k, v, b, h, dev):
    """Pointers, token count and shared strides of k and v [batch][n][heads][64] fp16 (0 for a dimension of one)."""
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise MmzError(f"{what}: k is a tensor [batch][n][heads][64]")
    n = k.shape[1]
    shape = (b, n, h, 64)
    for t, name in ((k, "k"), (v, "v")):
        if not (isinstance(t, torch.Tensor) and t.dtype is _F16 and t.shape == shape and t.get_device() == dev):
            _refuse(what, name, t, _F16, shape, dev)
    s = k.stride()
    if v.stride() != s or s[3] != 1:
        raise MmzError(f"{what}: k and v have the same strides, the last dimension dense")
    return k.data_ptr(), v.data_ptr(), n, _steps(s, shape)


def _steps(s, shape):
    return [t if n > 1 else 0 for t, n in zip(s, shape)]


def kv8_write(k, v, k8, v8, ks, vs, block=64, pos=None, stream=None):
    """Quantises the tokens k, v [b][n][heads][64] fp16 into the cache k8, v8 [b][heads][cap][64] (int8 or
    float8_e4m3fn) with the scales ks, vs [b][heads][ceil(cap / block)] float32, at positions pos[b].. (int32 [b]; None:
    from 0). A block that already has tokens keeps at least its scale; its codes are rounded again when it grows."""
    dev = _device("kv8_write", "k8", k8)
    b, h, cap, kind, c = _cache("kv8_write", k8, v8, ks, vs, block, dev)
    pk, pv, n, s = _pair("kv8_write", k, v, b, h, dev)
    at = _dense("kv8_write", "pos", pos, _I32, (b,), dev)
    _check(lib.mmz_kv8_write(pk, pv, s[0], s[1], s[2], *c, at, b, h, n, cap, block, kind, _stream(stream, dev)),
           "kv8_write")


def kv8_read(k8, v8, ks, vs, k, v, block=64, pos=None, lens=None, stream=None):
    """The cache's values at positions pos[b].. (None: from 0) into k, v [b][n][heads][64] fp16, zeros from position
    min(lens[b], cap) on (lens None: cap)."""
    dev = _device("kv8_read", "k8", k8)
    b, h, cap, kind, c = _cache("kv8_read", k8, v8, ks, vs, block, dev)
    pk, pv, n, s = _pair("kv8_read", k, v, b, h, dev)
    at, ln = _dense("kv8_read", "pos", pos, _I32, (b,), dev), _dense("kv8_read", "lens", lens, _I32, (b,), dev)
    _check(lib.mmz_kv8_read(*c, pk, pv, s[0], s[1], s[2], at, ln, b, h, n, cap, block, kind, _stream(stream, dev)),
           "kv8_read")


@functools.lru_cache(maxsize=256)
def attn8_scratch_bytes(batch, rows, q_heads, kv_heads, cap, slots=0):
    """Bytes of device scratch attn8 needs for such a call (0: none)."""
    return lib.mmz_attn8_scratch_bytes(batch, rows, q_heads, kv_heads, cap, slots)


def attn8(q, k8, v8, ks, vs, out, block=64, lens=None, causal=False, scale=0.125, probs=None, pslot=None, scratch=None,
          stream=None):
    """Attention of q [b][rows][q_heads][64] fp16 over the cache's first lens[b] positions (int32 [b]; None: all of
    them), into out of the same shape; causal: the rows are the sequence's last ones, row i sees lens - rows + i + 1
    positions. A row that sees nothing gives zeros. probs [b][slots][rows][cap] fp16 receives the probabilities of the
    heads with pslot[head] >= 0 (int32 [q_heads]). scratch: a uint8 tensor of attn8_scratch_bytes(...) (allocated here
    when None and needed)."""
    dev = _device("attn8", "k8", k8)
    b, h, cap, kind, c = _cache("attn8", k8, v8, ks, vs, block, dev)
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise MmzError("attn8: q is a tensor [batch][rows][q_heads][64]")
    shape = q.shape
    rows, hq = shape[1], shape[2]
    if shape[0] != b or shape[3] != 64:
        raise MmzError(f"attn8: q is {tuple(shape)}, not {(b, rows, hq, 64)}")
    pq, po = _strided("attn8", "q", q, _F16, shape, dev), _strided("attn8", "out", out, _F16, shape, dev)
    s, o = q.stride(), out.stride()
    if s[3] != 1 or o[3] != 1:
        raise MmzError("attn8: the last dimension of q and out is dense")
    s, o = _steps(s, shape), _steps(o, shape)
    ln = _dense("attn8", "lens", lens, _I32, (b,), dev)
    pp = ps = None
    slots = 0
    if probs is not None:
        slots = probs.shape[1] if isinstance(probs, torch.Tensor) and probs.dim() == 4 else 1
        pp = _dense("attn8", "probs", probs, _F16, (b, slots, rows, cap), dev)
        ps = _dense("attn8", "pslot", pslot, _I32, (hq,), dev)
    if scratch is None:
        need = attn8_scratch_bytes(b, rows, hq, h, cap, slots)
        if need:
            scratch = _own_scratch(need, q.device, stream)
    sp, sb = _scratch("attn8", scratch, dev)
    _check(lib.mmz_attn8(pq, s[0], s[1], s[2], *c, ln, po, o[0], o[1], o[2], b, rows, hq, h, cap, block, kind, causal,
                         scale, pp, ps, slots, sp, sb, _stream(stream, dev)), "attn8")


def _own_scratch(need, device, stream):
    """Scratch of one call: the allocator gives it to nobody else before the call's stream is through with it."""
    t = torch.empty(need, dtype=_U8, device=device)
    if stream is not None:
        t.record_stream(torch.cuda.ExternalStream(stream, device) if isinstance(stream, int) else stream)
    return t


def _scratch(what, t, dev):
    return (None, 0) if t is None else (_dense(what, "scratch", t, _U8, None, dev), t.numel())


def _outputs(what, rows, vocab, target, logp, entropy, lse, top_id, top_logp, sup, col, dev):
    """The arguments from sup to col: [rows] outputs, or [rows][steps] with a column counter."""
    if not isinstance(logp, torch.Tensor) or logp.dim() != (1 if col is None else 2):
        raise MmzError(f"{what}: logp is a tensor [rows], or [rows][steps] with col")
    ld = 1 if col is None else logp.shape[1]
    shape = (rows,) if col is None else (rows, ld)
    if col is not None and not (isinstance(col, torch.Tensor) and col.numel()):
        raise MmzError(f"{what}: col is an int32 tensor of one number")
    one = top_id if top_id is not None else top_logp
    top = one.shape[-1] if isinstance(one, torch.Tensor) and one.dim() else 0
    return (_dense(what, "sup", sup, _U8, (vocab,), dev), _dense(what, "target", target, _I32, shape, dev),
            _dense(what, "logp", logp, _F32, shape, dev), _dense(what, "entropy", entropy, _F32, shape, dev),
            _dense(what, "lse", lse, _F32, shape, dev), _dense(what, "top_id", top_id, _I32, shape + (top,), dev),
            _dense(what, "top_logp", top_logp, _F32, shape + (top,), dev), top, ld,
            _dense(what, "col", col, _I32, None, dev))


def token_logprobs(logits, target, logp, entropy=None, lse=None, top_id=None, top_logp=None, sup=None, col=None,
                   stream=None):
    """Per row of logits [rows][vocab] (fp16 or fp32): logp[r] = log p(target[r]), the entropy, log sum e^x, and the
    ids and log probabilities of the largest logits (top_id int32, top_logp float32 [rows][top <= 8]; ties to the lower
    id). sup [vocab] uint8: ids left out. With col (an int32 device scalar) target and outputs are [rows][steps] and
    column col[0] is read and written. A target outside the vocabulary has logp 0."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (_F16, _F32) or logits.dim() != 2:
        raise MmzError("token_logprobs: logits is an fp16 or fp32 tensor [rows][vocab]")
    dev = _device("token_logprobs", "logits", logits)
    rows, vocab = logits.shape
    px = _strided("token_logprobs", "logits", logits, logits.dtype, logits.shape, dev)
    s = logits.stride()
    if s[1] != 1 and vocab > 1:
        raise MmzError("token_logprobs: the last dimension of logits is dense")
    o = _outputs("token_logprobs", rows, vocab, target, logp, entropy, lse, top_id, top_logp, sup, col, dev)
    _check(lib.mmz_token_logprobs(px, s[0] if rows > 1 else vocab, logits.dtype is _F32, rows, vocab, *o,
                                  _stream(stream, dev)), "token_logprobs")


@functools.lru_cache(maxsize=256)
def linear_logprobs_scratch_bytes(rows, vocab, d):
    """Bytes of device scratch linear_logprobs needs for such a call."""
    return lib.mmz_linear_logprobs_scratch_bytes(rows, vocab, d)


def linear_logprobs(x, emb, target, logp, entropy=None, lse=None, top_id=None, top_logp=None, sup=None, col=None,
                    scratch=None, stream=None):
    """token_logprobs of the logits x . emb^T (x [rows][d], emb [vocab][d] fp16), in fp32 from the product on. scratch:
    a uint8 tensor of linear_logprobs_scratch_bytes(rows, vocab, d) (allocated here when None)."""
    what = "linear_logprobs"
    if not isinstance(x, torch.Tensor) or not isinstance(emb, torch.Tensor) or x.dim() != 2 or emb.dim() != 2:
        raise MmzError("linear_logprobs: x [rows][d] and emb [vocab][d] are tensors")
    dev = _device(what, "x", x)
    (rows, d), vocab = x.shape, emb.shape[0]
    px, pe = _strided(what, "x", x, _F16, x.shape, dev), _dense(what, "emb", emb, _F16, (vocab, d), dev)
    s = x.stride()
    if s[1] != 1:
        raise MmzError("linear_logprobs: the last dimension of x is dense")
    o = _outputs(what, rows, vocab, target, logp, entropy, lse, top_id, top_logp, sup, col, dev)
    if scratch is None:
        scratch = _own_scratch(linear_logprobs_scratch_bytes(rows, vocab, d), x.device, stream)
    sp, sb = _scratch(what, scratch, dev)
    _check(lib.mmz_linear_logprobs(px, s[0] if rows > 1 else d, pe, rows, vocab, d, *o, sp, sb, _stream(stream, dev)),
           what)
