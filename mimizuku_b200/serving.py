"""The 8-bit key/value cache (write, read back, attention) and the token log probabilities, over torch CUDA tensors.

Every call works on the current device and stream (or `stream`), checks its tensors on the host (MmzError) and returns
without waiting; outputs are tensors that the caller gives."""
import functools
import struct

import torch

from . import MmzError, _check, lib

_KIND = {torch.int8: 0, torch.float8_e4m3fn: 1}
_I32, _F16, _F32, _U8 = torch.int32, torch.float16, torch.float32, torch.uint8
_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice

# the argument structs of include/mimizuku_b200.h (native alignment: pointers and long long first, then the ints)
_KV8 = struct.Struct("4Q4q4i")
_ATTN8 = struct.Struct("Q3qQ3q5Q5if")
_LOGPROBS = struct.Struct("6QqQi4x")


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
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == dev):
        _refuse(what, name, t, dtype, shape, dev)
    return t.data_ptr()


def _dense(what, name, t, dtype, shape, dev):
    """The same of a contiguous one; 0 for None."""
    if t is None:
        return 0
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == dev
            and (shape is None or t.shape == shape) and t.is_contiguous()):
        _refuse(what, name, t, dtype, shape, dev)
    return t.data_ptr()


def _cache(what, k8, v8, ks, vs, block, dev):
    """(batch, heads, cap, mmz_kv8) of a cache."""
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
    return b, h, cap, _KV8.pack(k8.data_ptr(), v8.data_ptr(), ks.data_ptr(), vs.data_ptr(), cs[0] if b > 1 else 0,
                                cs[1] if h > 1 else 0, ss[0] if b > 1 else 0, ss[1] if h > 1 else 0, h, cap, block, kind)


def _pair(what, k, v, b, h, dev):
    """Pointers, shared strides (0 for a dimension of one) and token count of k and v [batch][n][heads][64] fp16."""
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
    return (k.data_ptr(), v.data_ptr(), s[0] if b > 1 else 0, s[1] if n > 1 else 0, s[2] if h > 1 else 0), n


def kv8_write(k, v, k8, v8, ks, vs, block=64, pos=None, stream=None):
    """Quantises the tokens k, v [b][n][heads][64] fp16 into the cache k8, v8 [b][heads][cap][64] (int8 or
    float8_e4m3fn) with the scales ks, vs [b][heads][ceil(cap / block)] float32, at positions pos[b].. (int32 [b]; None:
    from 0). A block that already has tokens keeps at least its scale; its codes are rounded again when it grows."""
    dev = _device("kv8_write", "k8", k8)
    b, h, cap, cache = _cache("kv8_write", k8, v8, ks, vs, block, dev)
    kv, n = _pair("kv8_write", k, v, b, h, dev)
    _check(lib.mmz_kv8_write(cache, *kv, _dense("kv8_write", "pos", pos, _I32, (b,), dev), b, n, _stream(stream, dev)),
           "kv8_write")


def kv8_read(k8, v8, ks, vs, k, v, block=64, pos=None, lens=None, stream=None):
    """The cache's values at positions pos[b].. (None: from 0) into k, v [b][n][heads][64] fp16, zeros from position
    min(lens[b], cap) on (lens None: cap)."""
    dev = _device("kv8_read", "k8", k8)
    b, h, cap, cache = _cache("kv8_read", k8, v8, ks, vs, block, dev)
    kv, n = _pair("kv8_read", k, v, b, h, dev)
    _check(lib.mmz_kv8_read(cache, *kv, _dense("kv8_read", "pos", pos, _I32, (b,), dev),
                            _dense("kv8_read", "lens", lens, _I32, (b,), dev), b, n, _stream(stream, dev)), "kv8_read")


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
    b, h, cap, cache = _cache("attn8", k8, v8, ks, vs, block, dev)
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise MmzError("attn8: q is a tensor [batch][rows][q_heads][64]")
    shape = q.shape
    qb, rows, hq, width = shape
    if qb != b or width != 64:
        raise MmzError(f"attn8: q is {tuple(shape)}, not {(b, rows, hq, 64)}")
    pq, po = _strided("attn8", "q", q, _F16, shape, dev), _strided("attn8", "out", out, _F16, shape, dev)
    s, o = q.stride(), out.stride()
    if s[3] != 1 or o[3] != 1:
        raise MmzError("attn8: the last dimension of q and out is dense")
    pp = ps = slots = 0
    if probs is not None:
        slots = probs.shape[1] if isinstance(probs, torch.Tensor) and probs.dim() == 4 else 1
        pp = _dense("attn8", "probs", probs, _F16, (b, slots, rows, cap), dev)
        ps = _dense("attn8", "pslot", pslot, _I32, (hq,), dev)
    sp = sb = 0
    if scratch is None:
        sb = attn8_scratch_bytes(b, rows, hq, h, cap, slots)
        if sb:
            scratch = _own_scratch(sb, q.device, stream)
            sp = scratch.data_ptr()
    else:
        sp, sb = _dense("attn8", "scratch", scratch, _U8, None, dev), scratch.numel()
    args = _ATTN8.pack(pq, s[0] if b > 1 else 0, s[1] if rows > 1 else 0, s[2] if hq > 1 else 0, po, o[0] if b > 1 else 0,
                       o[1] if rows > 1 else 0, o[2] if hq > 1 else 0, _dense("attn8", "lens", lens, _I32, (b,), dev), pp,
                       ps, sp, sb, b, rows, hq, slots, bool(causal), scale)
    _check(lib.mmz_attn8(cache, args, _stream(stream, dev)), "attn8")


def _own_scratch(need, device, stream):
    """Scratch of one call: the allocator gives it to nobody else before the call's stream is through with it."""
    t = torch.empty(need, dtype=_U8, device=device)
    if stream is not None:
        t.record_stream(torch.cuda.ExternalStream(stream, device) if isinstance(stream, int) else stream)
    return t


def _outputs(what, rows, target, logp, entropy, lse, top_id, top_logp, col, dev):
    """mmz_logprobs: [rows] outputs, or [rows][steps] with a column counter."""
    if not isinstance(logp, torch.Tensor) or logp.dim() != (1 if col is None else 2):
        raise MmzError(f"{what}: logp is a tensor [rows], or [rows][steps] with col")
    ld = 1 if col is None else logp.shape[1]
    shape = (rows,) if col is None else (rows, ld)
    if col is not None and not (isinstance(col, torch.Tensor) and col.numel()):
        raise MmzError(f"{what}: col is an int32 tensor of one number")
    one = top_id if top_id is not None else top_logp
    top = one.shape[-1] if isinstance(one, torch.Tensor) and one.dim() else 0
    return _LOGPROBS.pack(_dense(what, "target", target, _I32, shape, dev), _dense(what, "logp", logp, _F32, shape, dev),
                          _dense(what, "entropy", entropy, _F32, shape, dev), _dense(what, "lse", lse, _F32, shape, dev),
                          _dense(what, "top_id", top_id, _I32, shape + (top,), dev),
                          _dense(what, "top_logp", top_logp, _F32, shape + (top,), dev), ld,
                          _dense(what, "col", col, _I32, None, dev), top)


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
    s = logits.stride()
    if s[1] != 1 and vocab > 1:
        raise MmzError("token_logprobs: the last dimension of logits is dense")
    o = _outputs("token_logprobs", rows, target, logp, entropy, lse, top_id, top_logp, col, dev)
    _check(lib.mmz_token_logprobs(logits.data_ptr(), s[0] if rows > 1 else vocab, logits.dtype is _F32, rows, vocab,
                                  _dense("token_logprobs", "sup", sup, _U8, (vocab,), dev), o, _stream(stream, dev)),
           "token_logprobs")


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
    o = _outputs(what, rows, target, logp, entropy, lse, top_id, top_logp, col, dev)
    if scratch is None:
        sb = linear_logprobs_scratch_bytes(rows, vocab, d)
        scratch = _own_scratch(sb, x.device, stream)
        sp = scratch.data_ptr()
    else:
        sp, sb = _dense(what, "scratch", scratch, _U8, None, dev), scratch.numel()
    _check(lib.mmz_linear_logprobs(px, s[0] if rows > 1 else d, pe, rows, vocab, d,
                                   _dense(what, "sup", sup, _U8, (vocab,), dev), o, sp, sb, _stream(stream, dev)), what)
