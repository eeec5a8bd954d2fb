"""The 8-bit key/value cache (write, read back, attention) and the token log probabilities, over torch CUDA tensors.

Every call works on the current device and stream (or `stream`), checks its tensors on the host (MmzError) and returns
without waiting; outputs are tensors that the caller gives. The calls themselves are compiled (csrc/serving.cpp)."""
import torch  # noqa: F401  (its libraries, which the compiled calls link to)

from . import lib

try:
    from ._serving import attn8, kv8_read, kv8_write, linear_logprobs, token_logprobs  # noqa: F401
except ImportError as e:  # not there, or built for another torch or Python
    raise ImportError(f"mimizuku_b200/_serving.so does not load; build it with `python mimizuku_b200/build.py` ({e})") from e


def attn8_scratch_bytes(batch, rows, q_heads, kv_heads, cap, slots=0):
    """Bytes of device scratch attn8 needs for such a call (0: none)."""
    return lib.mmz_attn8_scratch_bytes(batch, rows, q_heads, kv_heads, cap, slots)


def linear_logprobs_scratch_bytes(rows, vocab, d):
    """Bytes of device scratch linear_logprobs needs for such a call."""
    return lib.mmz_linear_logprobs_scratch_bytes(rows, vocab, d)
