"""A paged key / value cache that is held in 4 bits: writing its pages, reading them back, attention over them, and copies of pages.

A page holds 64 tokens of one head of 64 or 128 elements (``uint8 [num_blocks, kv heads, page_bytes(dim)]`` for the keys and the same for the
values). Groups of 32 neighbouring elements of a token share two BF16 numbers, and an element stands for ``code * scale + lo``: ``lo`` is the
group's least element, ``scale`` its span / 15 rounded to BF16, a code is 0 .. 15, rounded to the nearest with ties to even. What an
element stands for is off by half a scale at most, and by the rounding of the scale (2^-8 of it for each step up to 15). That is 160 bytes a token and
head of 128 where BF16 pages take 512. Every token is quantised by itself, so rows may be taken back and written again, and pages may be copied. Elements are
2^15 at most; there is no least size, attention is as exact for small values as for others.

CUDA: ``csrc/kv4.cu``, ``csrc/attention_kv4.cu`` and ``csrc/attention_kv4_tc.cu``; the byte layout is in ``csrc/kv4.cuh``. CPU: the oracles below. Slots, block tables and lengths are
those of the BF16 cache (``ops.rope_kv_paged``, ``ops.attn_decode``, ``ops.attn_prefill``). Calls keep no state of their own and share no scratch: any stream may
be current, also one that is captured, as long as the tensors are on the current device."""
from __future__ import annotations

import ctypes
from ctypes import c_longlong

import torch

from . import BF16, _count, _require, ref
from .lib import KernelError, check, kernels, status_tensor

PAGE = 64
GROUP = 32
DIMS = (64, 128)
MOST = 2.0 ** 15                  # greatest magnitude of an element


def page_bytes(dim: int) -> int:
    """Bytes of a page of one head."""
    _require(dim in DIMS, "4-bit pages: heads of 64 or 128 elements")
    return PAGE * (dim // 2 + dim // 8)


def new_pages(num_blocks: int, hkv: int, dim: int, device) -> torch.Tensor:
    """Pages whose elements all stand for zero."""
    return torch.zeros(num_blocks, hkv, page_bytes(dim), dtype=torch.uint8, device=device)


# ------------------------------------------------------------------------------------------
# what the pages hold (oracles)
# ------------------------------------------------------------------------------------------
def _places(dim: int, keys: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Byte and shift of the code of every (token, element) of a page."""
    k, d = torch.meshgrid(torch.arange(PAGE), torch.arange(dim), indexing="ij")
    j, u, e = d // 32, d % 32 // 8, d % 8
    if keys:
        nibble = e // 2 + 4 * (e % 2)
        return k * (dim // 2) + 4 * (u * (dim // 32) + j) + nibble // 2, 4 * (nibble % 2)
    nibble, chunk = e // 2, 2 * u + e % 2
    row = k ^ (k // 8 % 2) if dim == 128 else k ^ (k // 4 % 4)
    chunk = chunk ^ (4 * (k // 4 % 2)) if dim == 128 else chunk
    return row * (dim // 2) + chunk * (dim // 16) + 2 * j + nibble // 2, 4 * (nibble % 2)


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes [..., dim] and (scale, lo) [..., dim / 32] of finite elements [..., dim], in 64 bits."""
    g = x.double().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1) + 0.0, g.amax(-1)                             # (no negative zero)
    m, e = torch.frexp((hi - lo) / 15)
    scale = torch.ldexp(torch.round(m * 256) / 256, e)
    scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
    code = torch.round((g - lo[..., None]) / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(0, 15)
    return torch.where(scale[..., None] > 0, code, 0.0).flatten(-2).to(torch.uint8), scale.to(BF16), lo.to(BF16)


def page_values(pages: torch.Tensor, dim: int, keys: bool) -> torch.Tensor:
    """What pages [blocks, heads, page_bytes] stand for: FP32 [blocks, heads, 64, dim]."""
    byte, shift = (t.to(pages.device) for t in _places(dim, keys))
    code = (pages[..., byte] >> shift.to(torch.uint8)) & 15
    stats = pages[..., PAGE * dim // 2:].contiguous().view(BF16).float().unflatten(-1, (PAGE, dim // GROUP, 2)).repeat_interleave(GROUP, dim=-2)
    return torch.addcmul(stats[..., 1], code.float(), stats[..., 0])


def token_bytes(dim: int, keys: bool) -> torch.Tensor:
    """Which bytes of a page each token has: int64 [64, page_bytes(dim) / 64], codes first (a byte's two codes belong to one token)."""
    codes = _places(dim, keys)[0].sort(dim=1).values[:, ::2]
    width = dim // GROUP * 4
    return torch.cat([codes, PAGE * dim // 2 + torch.arange(PAGE * width).view(PAGE, width)], dim=1)


def _write_rows(pages: torch.Tensor, rows: torch.Tensor, slots: torch.Tensor, dim: int, keys: bool) -> None:
    byte, shift = _places(dim, keys)
    code, scale, lo = quantise(rows)
    stats = torch.stack([scale, lo], dim=-1)
    for r, slot in enumerate(slots.tolist()):
        if slot < 0:
            continue
        block, k = divmod(slot, PAGE)
        page = pages[block]
        for even in (True, False):                                     # the two codes of a byte
            mine = shift[k] == (0 if even else 4)
            at = byte[k][mine]
            page[:, at] = (page[:, at] & (0xF0 if even else 0x0F)) | (code[r][:, mine] << (0 if even else 4))
        width = dim // GROUP * 4
        page[:, PAGE * dim // 2 + k * width: PAGE * dim // 2 + (k + 1) * width] = stats[r].flatten(1).contiguous().view(torch.uint8)


# ------------------------------------------------------------------------------------------
# arguments
# ------------------------------------------------------------------------------------------
# (plain ifs: a decode step makes these checks for every layer, and a message per check that holds costs more than the check)
def _check_pages(what: str, kpages: torch.Tensor, vpages: torch.Tensor, hkv: int, dim: int) -> int:
    if dim not in DIMS or hkv <= 0:
        raise KernelError(f"{what}: heads of 64 or 128 elements")
    shape = kpages.shape
    if kpages.dtype != torch.uint8 or vpages.dtype != torch.uint8 or vpages.shape != shape or not kpages.is_contiguous() or not vpages.is_contiguous() \
            or len(shape) != 3 or shape[0] == 0 or shape[1] != hkv or shape[2] != PAGE * (dim // 2 + dim // 8):
        raise KernelError(f"{what}: pages of keys and of values are uint8 [blocks, kv heads, page_bytes(dim)]")
    return shape[0]


def _check_device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            raise KernelError(f"{what}: tensors on one device")
    if device.type == "cuda" and device.index != _device():
        raise KernelError(f"{what}: tensors on the current device")


def _check_ints(what: str, n: int, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() != n:
            raise KernelError(f"{what}: int32 metadata, one number each")


# The current stream's handle and the current device as numbers: what torch.cuda.current_stream().cuda_stream and torch.cuda.current_device() give, without the 5 us
# of a stream object.
_raw_stream, _raw_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)


def _device() -> int:
    return torch.cuda.current_device() if _raw_device is None else _raw_device()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream if _raw_stream is None else _raw_stream(_device())


_bound: ctypes.CDLL | None = None


def _lib() -> ctypes.CDLL:
    """The kernels with the types of these launchers' arguments, so that numbers are passed as they are."""
    global _bound
    if _bound is None:
        lib = kernels()
        raw = getattr(lib, "_lib", lib)                                # (the checking build counts launches in front of it)
        p, i, n, f = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
        raw.ff_kv4_write.argtypes = [p, p, p, p, p, i, p, p, f, p, i, i, i, i, n, i, p, p]
        raw.ff_kv4_read.argtypes = [p, p, p, p, p, i, i, i, i, p, p]
        raw.ff_kv4_attn_rows.argtypes = [p, p, p, p, p, p, p, p, p, i, i, i, i, i, i, n, n, i, i, i, f, p, p]
        raw.ff_kv4_attn_tiles.argtypes = [p, p, p, p, p, p, p, p, p, i, i, i, i, i, i, n, n, i, i, i, f, p, p]
        raw.ff_copy_pages.argtypes = [p, p, i, p, p, i, p]
        _bound = lib
    return _bound


# ------------------------------------------------------------------------------------------
# writing and reading rows
# ------------------------------------------------------------------------------------------
def write_kv4(qkv: torch.Tensor, slots: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, hq: int, hkv: int, dim: int,
              cos_sin: torch.Tensor | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 0.0) -> torch.Tensor:
    """Packed BF16 rows ``[q heads | k heads | v heads]``: queries and keys are turned by ``cos_sin`` (``ops.rope_table``; float32 [rows, n, 2] of
    BF16 numbers, others are rounded to BF16; the first n elements of a head's halves turn), keys and values are written to ``slots`` (int32; page * 64 + place, below 0: not written). Returns the queries
    [rows, hq * dim]; ``qkv`` itself stays as it is (without ``cos_sin`` and norms the result is a view of it). ``q_norm`` / ``k_norm`` ([dim] BF16, given
    together): heads are RMS-normed with them and ``eps`` first. Rounds as ``ops.rope_kv_paged`` does. No two rows have the same slot. Keys and values that are
    not finite, or of magnitude above 2^15, raise the device status, and their group of 32 is stored as zeros."""
    blocks = _check_pages("write_kv4", kpages, vpages, hkv, dim)
    if qkv.dim() != 2 or qkv.stride(1) != 1 or qkv.dtype != BF16 or hq <= 0 or qkv.shape[1] < (hq + 2 * hkv) * dim:
        raise KernelError("write_kv4: packed BF16 rows with unit inner stride")
    rows, ld = qkv.shape[0], qkv.stride(0)
    if (q_norm is None) != (k_norm is None):
        raise KernelError("write_kv4: both head norms or none")
    _check_ints("write_kv4", rows, slots)
    if cos_sin is not None:
        _require(cos_sin.dtype == torch.float32 and cos_sin.dim() == 3 and cos_sin.shape[0] == rows and 0 < cos_sin.shape[1] <= dim // 2 and cos_sin.shape[2] == 2
                 and cos_sin.is_contiguous() and cos_sin.data_ptr() % 16 == 0, "write_kv4: cosines and sines float32 [rows, n, 2], aligned to 16 bytes")
    for w in (q_norm, k_norm):
        _require(w is None or (w.dtype == BF16 and w.numel() == dim and w.is_contiguous()), "write_kv4: head norms BF16 [dim]")
    _check_device("write_kv4", qkv, slots, kpages, vpages, cos_sin, q_norm, k_norm)
    plain = cos_sin is None and q_norm is None
    if not qkv.is_cuda:
        x = qkv[:, : (hq + 2 * hkv) * dim].reshape(rows, hq + 2 * hkv, dim)
        turned = x[:, : hq + hkv]
        if q_norm is not None:
            turned = torch.cat([ref.rmsnorm(turned[:, :hq], q_norm, eps), ref.rmsnorm(turned[:, hq:], k_norm, eps)], dim=1)
        if cos_sin is not None:
            n, half = cos_sin.shape[1], dim // 2
            r16 = lambda t: t.to(BF16).float()
            c, s = r16(cos_sin[:, None, :, 0]), r16(cos_sin[:, None, :, 1])
            turned = turned.float().clone()
            a, b = turned[..., :n].clone(), turned[..., half: half + n].clone()
            turned[..., :n] = r16(r16(a * c) - r16(b * s))
            turned[..., half: half + n] = r16(r16(b * c) + r16(a * s))
            turned = turned.to(BF16)
        k, v = turned[:, hq:], x[:, hq + hkv:]
        live = slots >= 0
        _require(bool((slots[live] < blocks * PAGE).all()), "write_kv4: a slot behind the last page")
        _require(all(bool((t[live].float().abs() <= MOST).all()) for t in (k, v)), "write_kv4: keys and values must be finite and at most 2^15")
        _write_rows(kpages, k, slots, dim, True)
        _write_rows(vpages, v, slots, dim, False)
        return qkv[:, : hq * dim] if plain else turned[:, :hq].reshape(rows, hq * dim)
    if (kpages.data_ptr() | vpages.data_ptr() | qkv.data_ptr()) % 16 or ld % 8:
        raise KernelError("write_kv4: rows and pages aligned to 16 bytes")
    q = qkv[:, : hq * dim] if plain else torch.empty(rows, hq * dim, dtype=BF16, device=qkv.device)
    if rows == 0:
        return q
    at = lambda t: None if t is None else t.data_ptr()
    check(_lib().ff_kv4_write(qkv.data_ptr(), slots.data_ptr(), kpages.data_ptr(), vpages.data_ptr(), at(cos_sin), 0 if cos_sin is None else cos_sin.shape[1], at(q_norm),
                              at(k_norm), eps, None if plain else q.data_ptr(), rows, hq, hkv, dim, ld, blocks, status_tensor(qkv.device).data_ptr(),
                              _stream()), "ff_kv4_write")
    _count()
    return q


def read_kv4(kpages: torch.Tensor, vpages: torch.Tensor, slots: torch.Tensor, dim: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of ``slots`` (int32 [rows]) as BF16 [rows, kv heads, dim]; rows of slots below 0 are zero."""
    _require(kpages.dim() == 3, "read_kv4: pages")
    hkv, rows = kpages.shape[1], slots.numel()
    blocks = _check_pages("read_kv4", kpages, vpages, hkv, dim)
    _check_ints("read_kv4", rows, slots)
    _check_device("read_kv4", kpages, vpages, slots)
    if not kpages.is_cuda:
        _require(bool((slots < blocks * PAGE).all()), "read_kv4: a slot behind the last page")
        at = slots.long().clamp(min=0)
        out = [page_values(p[at // PAGE], dim, keys)[torch.arange(rows), :, at % PAGE] for p, keys in ((kpages, True), (vpages, False))]
        return tuple(torch.where((slots >= 0)[:, None, None], t, 0.0).to(BF16) for t in out)
    if (kpages.data_ptr() | vpages.data_ptr()) % 16:
        raise KernelError("read_kv4: pages aligned to 16 bytes")
    k, v = (torch.empty(rows, hkv, dim, dtype=BF16, device=kpages.device) for _ in range(2))
    if rows:
        check(_lib().ff_kv4_read(kpages.data_ptr(), vpages.data_ptr(), slots.data_ptr(), k.data_ptr(), v.data_ptr(), rows, hkv, dim, blocks,
                                 status_tensor(kpages.device).data_ptr(), _stream()), "ff_kv4_read")
        _count()
    return k, v


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
def _check_attention(what, q, kpages, vpages, block_table, ctx_lens, hq, hkv, dim, scale, out) -> tuple[int, int]:
    blocks = _check_pages(what, kpages, vpages, hkv, dim)
    if q.dim() != 2 or q.stride(1) != 1 or q.dtype != BF16 or q.shape[1] < hq * dim:
        raise KernelError(f"{what}: BF16 rows of queries with unit inner stride")
    if hq <= 0 or hq % hkv:
        raise KernelError(f"{what}: a whole number of query heads per kv head")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous() or not 0 < block_table.shape[1] < 1 << 25:
        raise KernelError(f"{what}: int32 block table, positions of 31 bits")
    _check_ints(what, block_table.shape[0], ctx_lens)
    if not 0 < scale < float("inf"):
        raise KernelError(f"{what}: a positive scale")
    _check_device(what, q, kpages, vpages, block_table, ctx_lens, out)
    if out is not None and (out.shape != (q.shape[0], hq * dim) or out.dtype != BF16 or out.stride(1) != 1):
        raise KernelError(f"{what}: output BF16 [rows, hq * dim]")
    ldq = q.stride(0)
    if q.is_cuda:
        if (q.data_ptr() | kpages.data_ptr() | vpages.data_ptr()) % 16 or ldq % 8:
            raise KernelError(f"{what}: rows and pages aligned to 16 bytes")
        if out is not None and (out.data_ptr() % 16 or out.stride(0) % 8):
            raise KernelError(f"{what}: output rows aligned to 16 bytes")
    return ldq, blocks


def _attention_ref(q, kpages, vpages, block_table, q_start, q_lens, ctx_lens, hq, hkv, dim, scale, out):
    """In FP32 from the pages' values, rounded once."""
    res = torch.zeros(q.shape[0], hq, dim) if out is None else out.float().view(q.shape[0], hq, dim).clone()
    blocks = kpages.shape[0]
    for b in range(block_table.shape[0]):
        n, at, ctx = int(q_lens[b]), int(q_start[b]), int(ctx_lens[b])
        if n == 0:
            continue
        _require(0 <= at <= q.shape[0] - n, "attention over 4-bit pages: rows that the call does not have")
        _require(ctx <= block_table.shape[1] * PAGE, "attention over 4-bit pages: more keys than the block table has pages")
        res[at: at + n] = 0.0
        if ctx <= 0:
            continue
        pages = block_table[b, : (ctx + PAGE - 1) // PAGE].long()
        _require(bool(((pages >= 0) & (pages < blocks)).all()), "attention over 4-bit pages: a page outside the cache")
        k, v = (page_values(p[pages], dim, keys).transpose(0, 1).reshape(hkv, -1, dim)[:, :ctx] for p, keys in ((kpages, True), (vpages, False)))
        x = q[at: at + n, : hq * dim].float().view(n, hkv, hq // hkv, dim)
        score = torch.einsum("nhgd,hkd->hgnk", x, k) * scale
        hidden = torch.arange(ctx)[None, :] > torch.arange(ctx - n, ctx)[:, None]
        p = torch.softmax(score.masked_fill(hidden, float("-inf")), dim=-1).masked_fill(hidden.all(-1, keepdim=True), 0.0)
        res[at: at + n] = torch.einsum("hgnk,hkd->nhgd", p, v).reshape(n, hq, dim)
    res = res.view(q.shape[0], hq * dim).to(BF16)
    if out is None:
        return res
    out.copy_(res)
    return out


def in_tiles(max_q_len: int, hq: int, hkv: int) -> bool:
    """Whether attention of so many rows per sequence takes the kernel for prompts: FP16 tiles in shared memory for tcgen05 products of 128 rows, where
    the other one multiplies 8 or 16 rows by codes as they are. A sequence's rows times the query heads of a kv head are what counts: 24 sequences of up to 4000 tokens
    over 4 kv heads take 57 us with 32 such rows (58 in tiles), 65 in tiles with 80 (86); one of 30000 over 8 takes 38 with 32 (46), 46 in tiles with 64 (56). Contexts count too, and the
    rule leaves them out: a prompt of 37 rows with 4 heads each takes 14 either way, behind 1000 tokens 24 in tiles (20 as rows), behind 10000 34 (55); one of 100 rows alone 16 (14)."""
    return max_q_len * (hq // hkv) > 32


def _attention(q, ldq, kpages, vpages, blocks, block_table, q_start, q_lens, ctx_lens, nq, hq, hkv, dim, scale, max_ctx, out):
    batch, width, rows = block_table.shape[0], block_table.shape[1], q.shape[0]
    if out is None:
        out = torch.empty(rows, hq * dim, dtype=BF16, device=q.device)
    if batch == 0 or rows == 0:
        return out
    lib, floats = _lib(), c_longlong(0)
    most = width * PAGE if max_ctx is None else min(max_ctx, width * PAGE)
    tiles = in_tiles(nq, hq, hkv)
    if tiles:
        nsplit = lib.ff_kv4_tiles_plan(batch, rows, nq, hq, hkv, dim, most, ctypes.byref(floats))
    else:
        nsplit = lib.ff_kv4_attn_plan(batch, hq, hkv, nq, dim, most, ctypes.byref(floats))
        if q_start is not None and nsplit > 8:
            nsplit, floats.value = 8, 0
    scratch = torch.empty(floats.value, dtype=torch.float32, device=q.device) if floats.value else None
    tail = (hq, hkv, dim, ldq, out.stride(0), width, blocks, nsplit, scale, status_tensor(q.device).data_ptr(), _stream())
    head = (q.data_ptr(), kpages.data_ptr(), vpages.data_ptr(), block_table.data_ptr(), None if q_start is None else q_start.data_ptr(),
            None if q_lens is None else q_lens.data_ptr(), ctx_lens.data_ptr(), out.data_ptr(), None if scratch is None else scratch.data_ptr(), batch, rows, nq)
    if tiles:
        check(lib.ff_kv4_attn_tiles(*head, *tail), "ff_kv4_attn_tiles")
    else:
        check(lib.ff_kv4_attn_rows(*head, *tail), "ff_kv4_attn_rows")
    _count(1 if scratch is None else 3 if nsplit == 0 else 2)             # (a list of the work first, parts joined last)
    return out


def attn_decode_kv4(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor, ctx_lens: torch.Tensor, hq: int, hkv: int, dim: int,
                    scale: float, nq: int = 1, max_ctx: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``nq`` rows per sequence over 4-bit pages: ``q`` holds ``batch * nq`` BF16 rows (head h at columns ``h * dim``; it may be the packed rows),
    ``ctx_lens[b]`` counts the keys that the last of them sees, each row before it one less. Sequences of no keys give zeros. ``max_ctx``: most keys of a
    sequence (default: what the block table has room for); fixes how the work is split, and with it the result's last bits. Returns ``[batch * nq, hq * dim]``."""
    ldq, blocks = _check_attention("attn_decode_kv4", q, kpages, vpages, block_table, ctx_lens, hq, hkv, dim, scale, out)
    batch = block_table.shape[0]
    if nq <= 0 or q.shape[0] != batch * nq:
        raise KernelError("attn_decode_kv4: q rows must equal batch * nq")
    if not q.is_cuda:
        return _attention_ref(q, kpages, vpages, block_table, torch.arange(batch) * nq, [nq] * batch, ctx_lens, hq, hkv, dim, scale, out)
    return _attention(q, ldq, kpages, vpages, blocks, block_table, None, None, ctx_lens, nq, hq, hkv, dim, scale, max_ctx, out)


def attn_prefill_kv4(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor, q_lens: torch.Tensor,
                     ctx_lens: torch.Tensor, max_q_len: int, hq: int, hkv: int, dim: int, scale: float, max_ctx: int | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed rows over 4-bit pages: sequence b has the ``q_lens[b]`` rows from ``q_start[b]`` on (at most ``max_q_len``), the last of which
    sees ``ctx_lens[b]`` keys. A sequence with more rows than ``max_q_len``, or with rows that ``q`` does not have, raises the device status and gets nothing. Rows that belong to no sequence stay as they are in ``out`` (undefined without one). ``max_ctx`` as in :func:`attn_decode_kv4`.
    Returns ``[rows, hq * dim]``."""
    ldq, blocks = _check_attention("attn_prefill_kv4", q, kpages, vpages, block_table, ctx_lens, hq, hkv, dim, scale, out)
    _check_ints("attn_prefill_kv4", block_table.shape[0], q_start, q_lens)
    _check_device("attn_prefill_kv4", q, q_start, q_lens)
    if max_q_len <= 0:
        raise KernelError("attn_prefill_kv4: at least one row")
    if not q.is_cuda:
        _require(bool((q_lens <= max_q_len).all()), "attn_prefill_kv4: more rows of a sequence than max_q_len")
        return _attention_ref(q, kpages, vpages, block_table, q_start, q_lens, ctx_lens, hq, hkv, dim, scale, out)
    return _attention(q, ldq, kpages, vpages, blocks, block_table, q_start, q_lens, ctx_lens, max_q_len, hq, hkv, dim, scale, max_ctx, out)


# ------------------------------------------------------------------------------------------
# copies of pages
# ------------------------------------------------------------------------------------------
def copy_pages(tensors: list[torch.Tensor], src: list[int], dst: list[int]) -> None:
    """In every tensor (first dimension: pages; any type, widths may differ) page ``dst[i]`` becomes a copy of page ``src[i]``, in place. No page is
    written twice, and none that is written is read: those calls are refused. Keys and values of all layers go in one launch."""
    pairs = len(src)
    written = set(dst)
    if len(dst) != pairs or len(written) != pairs or not written.isdisjoint(src):
        raise KernelError("copy_pages: as many sources as destinations, and a page that is written is neither read nor written again")
    if pairs == 0 or not tensors:
        return
    where, least, most = tensors[0].get_device(), min(min(src), min(dst)), max(max(src), max(dst))
    base, size = [], []
    for t in tensors:
        n = t.shape[0] if t.dim() else 0
        if least < 0 or most >= n:
            raise KernelError("copy_pages: a page outside the cache")
        if t.get_device() != where or not t.is_contiguous():
            raise KernelError("copy_pages: contiguous tensors on one device")
        base.append(t.data_ptr())
        size.append(t.nbytes // n)
    if where < 0:
        a, b = torch.tensor(src), torch.tensor(dst)
        for t in tensors:
            t[b] = t[a]
        return
    if where != _device():
        raise KernelError("copy_pages: tensors on the current device")
    if any(v <= 0 or v % 16 for v in size) or any(v % 16 for v in base):
        raise KernelError("copy_pages: pages of whole 16 bytes")
    n = len(base)
    check(_lib().ff_copy_pages((ctypes.c_ulonglong * n)(*base), (c_longlong * n)(*size), n, (ctypes.c_int * pairs)(*src), (ctypes.c_int * pairs)(*dst), pairs,
                               _stream()), "ff_copy_pages")
    _count(-(-n // 160) * -(-pairs // 256))
