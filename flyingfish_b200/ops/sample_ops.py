"""Next tokens of a batch whose rows have settings of their own: temperature, top-k, top-p and min-p, drawn with a given random number per row. CUDA:
``csrc/sample.cu``; CPU: the oracle in 64 bits. Settings and numbers are data on the device, so a captured step serves any mix of them, greedy
rows included."""
from __future__ import annotations

from ctypes import c_int, c_longlong, c_void_p

import torch

from . import BF16, _count, _require, _rows2d, ref
from .lib import KernelError, check, kernels

F32, I32 = torch.float32, torch.int32


def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: torch.Tensor, top_k: torch.Tensor | None = None,
                  top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  probs: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``logits`` [rows, vocab] BF16 or FP32; ``uniforms`` (in [0, 1)), ``temperature``, ``top_p``, ``min_p`` FP32 and ``top_k`` int32, one per row. Returns the
    drawn ids (int32) and the probability each had among what was left to draw from (FP32).

    Tokens are ordered by logit, the larger first, equal ones by id. A row keeps the least of: its first ``top_k`` tokens (all where that is 0 or less); the
    smallest prefix whose mass reaches ``top_p`` of the whole mass of ``softmax(logits / temperature)`` (all from 1 on, one token at 0 or less); the tokens of
    at least ``min_p`` times the largest probability (all at 0 or less, those of the largest from 1 on). Drawn is the lowest id whose sum of kept masses up to it
    passes ``uniforms`` times their sum. ``temperature`` 0 or less: the lowest id of the largest logit, probability 1. NaN logits count as -inf, which is
    never drawn, and +inf shares everything among its equals; a row of -inf gives id 0 with probability 0. On a GPU masses are sums in 64 bits of weights that
    are held to 1.2e-12 of themselves, so the ids are the definition's unless a border lies within a few 1e-12 of the mass from where a token begins or ends; a
    weight below 2^-1000 of the largest counts as none, everywhere. The settings do not follow one another: ``top_p`` is a share of the mass before ``top_k`` and ``min_p``
    cut anything off. On a GPU a row lies in the shared memory of 8 multiprocessors: 380 thousand FP32 tokens or 760 thousand BF16
    ones, and there are 65535 rows at most."""
    rows, ld = _rows2d(logits)
    at = logits.get_device()
    vocab = logits.shape[1]
    _require(logits.dtype in (BF16, F32) and vocab > 0, "sample_tokens: bf16 or fp32 logits")
    _require(vocab < 1 << 31, "sample_tokens: ids are 32 bits wide")
    for t, dtype, name in ((uniforms, F32, "uniforms"), (temperature, F32, "temperature"), (top_k, I32, "top_k"), (top_p, F32, "top_p"), (min_p, F32, "min_p"),
                           (out, I32, "out"), (probs, F32, "probs")):
        if t is not None and not (t.dtype == dtype and t.dim() == 1 and t.shape[0] == rows and t.is_contiguous() and t.get_device() == at):
            raise KernelError(f"sample_tokens: {name} is one {dtype} per row on the logits' device")
    if not logits.is_cuda:
        ids, p = ref.sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p)
        return (ids if out is None else out.copy_(ids)), (p if probs is None else probs.copy_(p))
    _require(at == torch.cuda.current_device(), "sample_tokens: operands on another device than the current one")
    if out is None:
        out = logits.new_empty(rows, dtype=I32)
    if probs is None:
        probs = logits.new_empty(rows, dtype=F32)
    if rows == 0:
        return out, probs
    rc = _launcher()(logits.data_ptr(), logits.dtype == F32, uniforms.data_ptr(), temperature.data_ptr(), _at(top_k), _at(top_p), _at(min_p), out.data_ptr(),
                     probs.data_ptr(), rows, vocab, ld, torch._C._cuda_getCurrentRawStream(at))
    check(rc, "ff_sample_tokens")
    _count()
    return out, probs


def _at(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_typed = None


def _launcher():
    """``ff_sample_tokens`` with its argument types declared: plain numbers are converted by the call."""
    global _typed
    if _typed is None:
        fn = kernels().ff_sample_tokens
        if hasattr(fn, "argtypes"):                   # the checking build wraps the function
            fn.argtypes = [c_void_p, c_int] + [c_void_p] * 7 + [c_int, c_int, c_longlong, c_void_p]
            _typed = fn
        else:
            return lambda *v: fn(*(c_void_p(q) if i in (0, 2, 3, 4, 5, 6, 7, 8, 12) else c_longlong(q) if i == 11 else int(q) for i, q in enumerate(v)))
    return _typed
