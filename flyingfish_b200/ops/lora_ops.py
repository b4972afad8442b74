"""Low-rank adapters of many requests beside a shared projection: ``y = x W^T`` plus, for a row with an adapter, ``scale (x A^T) B^T`` of
that adapter, rounded once. The rows of a batch have an adapter each or none; which ones is data on the device, so a captured step serves
any mix. CUDA: ``csrc/lora.cu`` (BF16, FP32 sums) with the products of ``csrc/gemm_skinny.cu`` and ``csrc/gemm_bf16.cu``; CPU: FP32 oracle.

The adapters of one projection form an :class:`AdapterStack` (:func:`pack_stack` builds one, once). A stack's weights are taken to be finite
where they are within an adapter's rank; what is not reaches the rows of that adapter only. As with ``ops.linear``, weights (a stack's among them) may be
read ahead of what the stream still holds, and calls of up to 128 rows use the device's workspace: one stream at a time, or a ``SideLane``."""
from __future__ import annotations

import ctypes
import itertools
import os
from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import NamedTuple

import torch

from . import BF16, SKINNY_MAX_M, _count, _require, _rows2d, ref, rope_in_product, rope_kv_paged, rope_table, silu_mul_interleaved, workspace
from .lib import KernelError, check, kernels, status_tensor

_calls = itertools.count(int.from_bytes(os.urandom(8), "little") | 1 << 62)          # numbers of calls: what a word of memory does not hold by chance
MAX_RANK = 1024                  # rank rows of a stack, all parts of a fused projection together
GATES = (0, 3, 5)                # gates that the products' epilogues know (ops.linear_swiglu)


class AdapterStack(NamedTuple):
    """The adapters of one projection ``[N, K]``. ``a`` [adapters, R, K] and ``b`` [adapters, N, R] are BF16, ``scale`` FP32 [adapters], or [adapters, R]
    where an adapter's rank rows have scales of their own; R is a multiple of 16 and the rank rows behind an adapter's own are zero. ``ranks`` (int32 [adapters]) says how many rows that are, so that the rest is
    not read. ``part_of`` (int32 [N / 64]), ``parts`` and ``step`` describe a fused projection: its adapters' ranks come in steps of ``step`` (16 or 32), step s
    belongs to part ``s % parts``, and the 64 columns from ``64 i`` have non-zero ``b`` in the steps of part ``part_of[i]`` only."""
    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor
    ranks: torch.Tensor | None = None
    part_of: torch.Tensor | None = None
    parts: int = 1
    step: int = 16

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.a, self.b, self.scale, self.ranks, self.part_of) if t is not None)


def pack_stack(adapters: list[list[tuple[torch.Tensor, torch.Tensor, float] | None]], k: int, columns: list[int], device,
               dtype: torch.dtype = BF16, interleave: bool = False) -> AdapterStack:
    """``adapters``: for every adapter one entry per part of the projection (one part, or those of a fused one, ``columns`` wide each): ``(A [r, K],
    B [columns, r], scale)`` or None where the adapter leaves the part alone. ``interleave``: two parts whose columns lie in turns of 64 (gate and up).
    A part's scale is a number, or a tensor of one per rank. Neither matrix takes a scale into itself: with different ones the stack has a scale per rank row."""
    parts, n = len(columns), sum(columns)
    _require(bool(adapters) and all(len(p) == parts for p in adapters), "pack_stack: an entry per part for every adapter")
    _require(not interleave or (parts == 2 and columns[0] == columns[1] and columns[0] % 64 == 0), "pack_stack: two equal parts interleave")
    _require(parts == 1 or all(c % 64 == 0 for c in columns), "pack_stack: parts of whole 64 columns")
    most = max((e[0].shape[0] for p in adapters for e in p if e is not None), default=0)
    step = 16 if most <= 16 else 32
    r = max(1, (most + step - 1) // step) * step * parts
    _require(r <= MAX_RANK, f"pack_stack: ranks of {parts} parts of {most} exceed {MAX_RANK}")
    a = torch.zeros(len(adapters), r, k, dtype=dtype)
    b = torch.zeros(len(adapters), n, r, dtype=dtype)
    scale, ranks = torch.ones(len(adapters)), torch.zeros(len(adapters), dtype=torch.int32)
    scales, alike = torch.ones(len(adapters), r), True           # alike: every adapter's parts have one scale
    for i, entry in enumerate(adapters):
        at, own = 0, []
        for j, part in enumerate(entry):
            if part is not None:
                pa, pb, s = part
                rank = pa.shape[0]
                _require(pa.shape == (rank, k) and pb.shape == (columns[j], rank), f"pack_stack: adapter {i}: A [{rank}, {k}] and B [{columns[j]}, {rank}]")
                pa, pb = pa.to("cpu", dtype), pb.to("cpu", dtype)
                _require(bool(torch.isfinite(pa).all()) and bool(torch.isfinite(pb).all()), f"pack_stack: adapter {i} holds infinities or NaN")
                where = torch.tensor([(q // step * parts + j) * step + q % step for q in range(rank)], dtype=torch.long)
                a[i, where], b[i, at: at + columns[j], where] = pa, pb
                scales[i, where] = torch.as_tensor(s, dtype=torch.float32)
                own.append(scales[i, where])
                ranks[i] = max(int(ranks[i]), (rank + step - 1) // step * step * parts)
            at += columns[j]
        own = torch.cat([*own, torch.empty(0)])
        if own.numel():
            scale[i], alike = own[0], alike and bool((own == own[0]).all())
    part_of = None
    if interleave:
        b = b.view(len(adapters), 2, n // 128, 64, r).transpose(1, 2).reshape(len(adapters), n, r).contiguous()
        part_of = torch.arange(n // 64, dtype=torch.int32) % 2
    elif parts > 1:
        part_of = torch.repeat_interleave(torch.arange(parts, dtype=torch.int32), torch.tensor([c // 64 for c in columns]))
    move = lambda t: None if t is None else t.to(device)
    return AdapterStack(move(a), move(b), move(scale if alike else scales), move(ranks), move(part_of), parts, step)


class _Lora(ctypes.Structure):            # FfLora of csrc/lora.cu
    _fields_ = [(n, c_void_p) for n in ("x", "w", "y", "a", "b", "scale", "ranks", "ids", "part_of", "t", "scratch", "counters", "status", "cos_sin",
                                        "slots", "kcache", "vcache")] + [("scratch_bytes", c_longlong), ("counter_bytes", c_longlong), ("call", c_longlong)] + \
               [(n, c_int) for n in ("M", "N", "K", "ldx", "ldw", "ldy", "R", "adapters", "parts", "step", "epi", "gate", "scales")] + [("limit", c_float)] + \
               [(n, c_int) for n in ("hq", "hkv", "rot_dim", "block_size", "num_blocks")]


def _check_stack(x: torch.Tensor, n: int, stack: AdapterStack, ids: torch.Tensor) -> tuple[int, int]:
    """(adapters, R) of a stack that fits the projection."""
    a, b, scale, ranks, part_of, parts, step = stack
    _require(a.dim() == 3 and b.dim() == 3 and a.shape[2] == x.shape[1], "adapters: A [adapters, R, K] of the projection's K")
    count, r = a.shape[0], a.shape[1]
    _require(b.shape == (count, n, r) and scale.shape in ((count,), (count, r)), "adapters: B [adapters, N, R], a scale per adapter or rank row")
    _require(count > 0 and 0 < r <= MAX_RANK and r % 16 == 0, f"adapters: R is a multiple of 16, at most {MAX_RANK}")
    _require(a.dtype == b.dtype == x.dtype and scale.dtype == torch.float32, "adapters: weights of the operands' type, FP32 scales")
    _require(a.is_contiguous() and b.is_contiguous() and scale.is_contiguous(), "adapters: contiguous weights")
    _require(ids.dtype == torch.int32 and ids.shape == (x.shape[0],) and ids.is_contiguous(), "adapters: one int32 id per row")
    _require(ranks is None or (ranks.dtype == torch.int32 and ranks.shape == (count,) and ranks.is_contiguous()), "adapters: int32 ranks")
    _require(part_of is None or (part_of.dtype == torch.int32 and part_of.numel() * 64 >= n and part_of.is_contiguous() and parts > 0 and step in (16, 32) and r % step == 0),
             "adapters: int32 parts, ranks in whole steps")
    return count, r


def _at(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _run(x: torch.Tensor, w: torch.Tensor, stack: AdapterStack, ids: torch.Tensor, out: torch.Tensor | None, width: int, epi: int, gate: int = 0,
         limit: float = 0.0, rope: tuple | None = None) -> torch.Tensor:
    _require(isinstance(w, torch.Tensor) and x.dtype == w.dtype == BF16, "linear_lora: BF16 operands required on CUDA")
    m, ldx = _rows2d(x)
    n, ldw = _rows2d(w)
    k = x.shape[1]
    _require(w.shape[1] == k, "linear_lora: inner dimensions differ")
    count, r = _check_stack(x, n, stack, ids)
    a, b, scale, ranks, part_of, parts, step = stack
    at = x.get_device()
    _require(at == torch.cuda.current_device(), "linear_lora: operands on another device than the current one")
    _require(at == w.get_device() == a.get_device() == b.get_device() == scale.get_device() == ids.get_device() and
             (ranks is None or ranks.get_device() == at) and (part_of is None or part_of.get_device() == at) and (out is None or out.get_device() == at),
             "linear_lora: operands on several devices")
    if out is None:
        out = x.new_empty(m, width)
    else:
        _require(out.shape == (m, width) and out.stride(1) == 1 and out.dtype == BF16, "linear_lora: bad output tensor")
    if m == 0:
        return out
    dev = x.device
    t, call = x.new_empty(m * 2 * r + 4), next(_calls) & (1 << 63) - 1          # of this call alone
    ws = workspace(dev)
    cs, slots, kc, vc, heads = rope if rope is not None else (None, None, None, None, (0, 0, 0, 0, 0))
    lib, stream = kernels(), c_void_p(torch._C._cuda_getCurrentRawStream(at))
    for attempt in (0, 1):
        form = _Lora(x.data_ptr(), w.data_ptr(), out.data_ptr(), a.data_ptr(), b.data_ptr(), scale.data_ptr(), _at(ranks), ids.data_ptr(), _at(part_of), t.data_ptr(),
                     ws.gemm_scratch.data_ptr(), ws.gemm_counters.data_ptr(), status_tensor(dev).data_ptr(), _at(cs), _at(slots), _at(kc), _at(vc),
                     ws.gemm_scratch.numel() * 4, ws.gemm_counters.numel() * 4, call, m, n, k, ldx, ldw, out.stride(0), r, count, parts, step, epi, gate, scale.dim() - 1, limit, *heads)
        rc = lib.ff_linear_lora(ctypes.byref(form), stream)
        if rc != -5 or attempt or m > SKINNY_MAX_M:
            break
        scratch_b, counter_b = c_longlong(0), c_longlong(0)          # the product's scratch is too small: nothing was launched
        plan = (m, n, k) if not epi else (m, n, k, epi)
        (lib.ff_gemm_skinny_plan_epi if epi else lib.ff_gemm_skinny_plan)(*plan, ctypes.byref(scratch_b), ctypes.byref(counter_b))
        ws.ensure("gemm_scratch", scratch_b.value // 4)
        _require(counter_b.value // 4 <= ws.gemm_counters.numel(), "linear_lora: too many column tiles for counters")
    check(rc, "ff_linear_lora")
    _count(2)
    return out


def linear_lora(x: torch.Tensor, w: torch.Tensor, stack: AdapterStack, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`ops.linear` (BF16 result) with the adapter ``ids[row]`` (int32; negative: none) of ``stack`` added to every row before the sums are rounded. Rows
    without an adapter have the bits of ``ops.linear``, and a row's bits do not depend on the other rows' adapters. An id past the stack raises the status word
    (bounds) and counts as none."""
    if not x.is_cuda:
        _check_stack(x, w.shape[0], stack, ids)
        y = ref.linear_lora(x, w, stack.a, stack.b, stack.scale, ids)
        return y if out is None else out.copy_(y)
    return _run(x, w, stack, ids, out, w.shape[0], 0)


def linear_swiglu_lora(x: torch.Tensor, w_interleaved: torch.Tensor, stack: AdapterStack, ids: torch.Tensor, out: torch.Tensor | None = None,
                       mode: int = 0, limit: float = 0.0) -> torch.Tensor:
    """:func:`ops.linear_swiglu` with adapters on the gate and up projections (``b`` rows in the weight's interleaved order)."""
    if not x.is_cuda or mode not in GATES:
        return silu_mul_interleaved(linear_lora(x, w_interleaved, stack, ids), out, mode, limit)
    _require(w_interleaved.shape[0] % 256 == 0, "linear_swiglu_lora: N must be a multiple of 256")
    return _run(x, w_interleaved, stack, ids, out, w_interleaved.shape[0] // 2, 1, mode, limit)


def linear_rope_kv_lora(x: torch.Tensor, wqkv: torch.Tensor, stack: AdapterStack, ids: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                        kcache: torch.Tensor, vcache: torch.Tensor, hq: int, hkv: int, dim: int, theta: float, cos_sin: torch.Tensor | None = None
                        ) -> torch.Tensor:
    """:func:`ops.linear_rope_kv` with adapters on the q, k and v projections: heads of 128 turn and go to the cache in the product's epilogue where
    :func:`ops.rope_in_product` says so, others in a kernel of their own."""
    if not x.is_cuda or dim != 128 or not rope_in_product(x.shape[0], wqkv.shape[0], x.shape[1]):
        qkv = linear_lora(x, wqkv, stack, ids)
        rope_kv_paged(qkv, positions, slots, kcache, vcache, hq, hkv, dim, theta)
        return qkv
    rows, n = x.shape[0], wqkv.shape[0]
    _require(positions.dtype == slots.dtype == torch.int32 and positions.shape == slots.shape == (rows,) and slots.is_contiguous(), "linear_rope_kv_lora: int32 metadata")
    nb, ch, bs, cd = kcache.shape
    _require(ch == hkv and cd == dim and vcache.shape == kcache.shape and n == (hq + 2 * hkv) * 128, "linear_rope_kv_lora: cache geometry differs from the heads")
    _require(kcache.is_contiguous() and vcache.is_contiguous() and kcache.dtype == vcache.dtype == BF16, "linear_rope_kv_lora: cache layout")
    _require(all(t.device == x.device for t in (positions, slots, kcache, vcache)), "linear_rope_kv_lora: operands on several devices")
    if rows and cos_sin is None:
        cos_sin = rope_table(positions, dim, theta)
    if rows:
        _require(cos_sin.shape == (rows, dim // 2, 2) and cos_sin.dtype == torch.float32 and cos_sin.is_contiguous() and cos_sin.device == x.device,
                 "linear_rope_kv_lora: cos/sin table")
    return _run(x, wqkv, stack, ids, None, n, 2, rope=(cos_sin, slots, kcache, vcache, (hq, hkv, dim, bs, nb)))
