"""A paged key / value cache that is held in 4 bits: writing its pages, reading them back, attention over them, and copies of pages.

A page holds 64 tokens of one head of 64 or 128 elements (``uint8 [num_blocks, kv heads, page_bytes(dim)]`` for the keys and the same for the
values). Groups of 32 neighbouring elements of a token share two BF16 numbers, and an element stands for ``code * scale + lo``: ``lo`` is the
group's least element, ``scale`` its span / 15 rounded to BF16, a code is 0 .. 15, rounded to the nearest with ties to even. What an
element stands for is off by half a scale at most, and by the rounding of the scale (2^-8 of it for each step up to 15). That is 160 bytes a token and
head of 128 where BF16 pages take 512. Every token is quantised by itself, so rows may be taken back and written again, and pages may be copied.

CUDA: ``csrc/kv4.cu`` and ``csrc/attention_kv4.cu``; the byte layout is in ``csrc/kv4.cuh``. CPU: the oracles below. Slots, block tables and lengths are
those of the BF16 cache (``ops.rope_kv_paged``, ``ops.attn_decode``, ``ops.attn_prefill``). Calls keep no state of their own and share no scratch: any stream may
be current, also one that is captured, as long as the tensors are on the current device."""
from __future__ import annotations

import ctypes
from ctypes import c_float, c_longlong

import torch

from . import BF16, _count, _require, _rows2d, ref
from .lib import KernelError, check, kernels, ptr, status_tensor, stream_ptr

PAGE = 64
GROUP = 32
DIMS = (64, 128)
MOST = 2.0 ** 15                  # greatest magnitude of an element: FP16 holds it


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
    lo, hi = g.amin(-1), g.amax(-1)
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
def _check_pages(what: str, kpages: torch.Tensor, vpages: torch.Tensor, hkv: int, dim: int) -> int:
    _require(dim in DIMS, f"{what}: heads of 64 or 128 elements")
    for t in (kpages, vpages):
        _require(t.dtype == torch.uint8 and t.dim() == 3 and t.is_contiguous() and t.shape[1] == hkv and t.shape[2] == page_bytes(dim),
                 f"{what}: pages are uint8 [blocks, kv heads, page_bytes(dim)]")
    _require(kpages.shape[0] == vpages.shape[0] > 0, f"{what}: as many pages of keys as of values")
    return kpages.shape[0]


def _check_device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    _require(all(t is None or t.device == first.device for t in others), f"{what}: tensors on one device")
    if first.is_cuda:
        _require(first.device.index == torch.cuda.current_device(), f"{what}: tensors on the current device")


def _check_ints(what: str, n: int, *tensors: torch.Tensor) -> None:
    for t in tensors:
        _require(t.dtype == torch.int32 and t.is_contiguous() and t.numel() == n, f"{what}: int32 metadata, one number each")


# ------------------------------------------------------------------------------------------
# writing and reading rows
# ------------------------------------------------------------------------------------------
def write_kv4(qkv: torch.Tensor, slots: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, hq: int, hkv: int, dim: int,
              cos_sin: torch.Tensor | None = None, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 0.0) -> torch.Tensor:
    """Packed BF16 rows ``[q heads | k heads | v heads]``: queries and keys are turned by ``cos_sin`` (``ops.rope_table``; float32 [rows, n, 2], the
    first n elements of a head's halves turn), keys and values are written to ``slots`` (int32; page * 64 + place, below 0: not written). Returns the queries
    [rows, hq * dim]; ``qkv`` itself stays as it is (without ``cos_sin`` and norms the result is a view of it). ``q_norm`` / ``k_norm`` ([dim] BF16, given
    together): heads are RMS-normed with them and ``eps`` first. Rounds as ``ops.rope_kv_paged`` does. No two rows have the same slot. Keys and values that are
    not finite, or of magnitude above 2^15, raise the device status, and their group of 32 is stored as zeros."""
    rows, ld = _rows2d(qkv)
    blocks = _check_pages("write_kv4", kpages, vpages, hkv, dim)
    _require(hq > 0 and hkv > 0 and qkv.shape[1] >= (hq + 2 * hkv) * dim and qkv.dtype == BF16, "write_kv4: packed BF16 rows")
    _require((q_norm is None) == (k_norm is None), "write_kv4: both head norms or none")
    _check_ints("write_kv4", rows, slots)
    if cos_sin is not None:
        _require(cos_sin.dtype == torch.float32 and cos_sin.dim() == 3 and cos_sin.shape[0] == rows and 0 < cos_sin.shape[1] <= dim // 2 and cos_sin.shape[2] == 2
                 and cos_sin.is_contiguous(), "write_kv4: cosines and sines float32 [rows, n, 2]")
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
            c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
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
    _require(kpages.data_ptr() % 16 == 0 and vpages.data_ptr() % 16 == 0 and qkv.data_ptr() % 16 == 0 and ld % 8 == 0, "write_kv4: rows and pages aligned to 16 bytes")
    q = qkv[:, : hq * dim] if plain else torch.empty(rows, hq * dim, dtype=BF16, device=qkv.device)
    if rows == 0:
        return q
    rc = kernels().ff_kv4_write(ptr(qkv), ptr(slots), ptr(kpages), ptr(vpages), ptr(cos_sin), 0 if cos_sin is None else cos_sin.shape[1], ptr(q_norm), ptr(k_norm),
                                c_float(eps), ptr(None if plain else q), rows, hq, hkv, dim, c_longlong(ld), blocks, ptr(status_tensor(qkv.device)), stream_ptr())
    check(rc, "ff_kv4_write")
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
    _require(kpages.data_ptr() % 16 == 0 and vpages.data_ptr() % 16 == 0, "read_kv4: pages aligned to 16 bytes")
    k, v = (torch.empty(rows, hkv, dim, dtype=BF16, device=kpages.device) for _ in range(2))
    if rows:
        check(kernels().ff_kv4_read(ptr(kpages), ptr(vpages), ptr(slots), ptr(k), ptr(v), rows, hkv, dim, blocks, ptr(status_tensor(kpages.device)), stream_ptr()),
              "ff_kv4_read")
        _count()
    return k, v


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------
def _check_attention(what: str, q, kpages, vpages, block_table, ctx_lens, hq, hkv, dim, scale, out) -> tuple[int, int, int]:
    rows, ldq = _rows2d(q)
    blocks = _check_pages(what, kpages, vpages, hkv, dim)
    _require(hkv > 0 and hq % hkv == 0 and hq > 0, f"{what}: a whole number of query heads per kv head")
    _require(q.dtype == BF16 and q.shape[1] >= hq * dim, f"{what}: BF16 queries")
    _require(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.is_contiguous() and block_table.shape[1] > 0, f"{what}: int32 block table")
    _require(block_table.shape[1] < 1 << 25, f"{what}: positions of 31 bits")
    _check_ints(what, block_table.shape[0], ctx_lens)
    _require(scale > 0, f"{what}: a positive scale")
    _check_device(what, q, kpages, vpages, block_table, ctx_lens, out)
    if out is not None:
        _require(out.shape == (rows, hq * dim) and out.dtype == BF16 and out.stride(1) == 1, f"{what}: output BF16 [rows, hq * dim]")
    if q.is_cuda:
        _require(q.data_ptr() % 16 == 0 and ldq % 8 == 0 and kpages.data_ptr() % 16 == 0 and vpages.data_ptr() % 16 == 0, f"{what}: rows and pages aligned to 16 bytes")
    return rows, ldq, blocks


def _attention_ref(q, kpages, vpages, block_table, q_start, q_lens, ctx_lens, hq, hkv, dim, scale, out):
    """In FP32 from the pages' values, rounded once."""
    res = torch.zeros(q.shape[0], hq, dim) if out is None else out.float().view(q.shape[0], hq, dim).clone()
    blocks = kpages.shape[0]
    for b in range(block_table.shape[0]):
        n, at, ctx = int(q_lens[b]), int(q_start[b]), int(ctx_lens[b])
        if n == 0:
            continue
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
        p = torch.softmax(score.masked_fill(hidden, float("-inf")), dim=-1).nan_to_num(0.0)
        res[at: at + n] = torch.einsum("hgnk,hkd->nhgd", p, v).reshape(n, hq, dim)
    res = res.view(q.shape[0], hq * dim).to(BF16)
    if out is None:
        return res
    out.copy_(res)
    return out


def attn_decode_kv4(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor, ctx_lens: torch.Tensor, hq: int, hkv: int, dim: int,
                    scale: float, nq: int = 1, max_ctx: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of ``nq`` rows per sequence over 4-bit pages: ``q`` holds ``batch * nq`` BF16 rows (head h at columns ``h * dim``; it may be the packed rows),
    ``ctx_lens[b]`` counts the keys that the last of them sees, each row before it one less. Sequences of no keys give zeros. ``max_ctx``: most keys of a
    sequence (default: what the block table has room for); fixes how the work is split, and with it the result's last bits. Returns ``[batch * nq, hq * dim]``."""
    rows, ldq, blocks = _check_attention("attn_decode_kv4", q, kpages, vpages, block_table, ctx_lens, hq, hkv, dim, scale, out)
    batch = block_table.shape[0]
    _require(nq > 0 and rows == batch * nq, "attn_decode_kv4: q rows must equal batch * nq")
    if not q.is_cuda:
        return _attention_ref(q, kpages, vpages, block_table, torch.arange(batch) * nq, [nq] * batch, ctx_lens, hq, hkv, dim, scale, out)
    if out is None:
        out = torch.empty(rows, hq * dim, dtype=BF16, device=q.device)
    if batch == 0:
        return out
    width = block_table.shape[1]
    lib = kernels()
    floats = c_longlong(0)
    nsplit = lib.ff_kv4_attn_plan(batch, hq, hkv, nq, dim, min(max_ctx or width * PAGE, width * PAGE), ctypes.byref(floats))
    scratch = torch.empty(floats.value, dtype=torch.float32, device=q.device) if floats.value else None
    rc = lib.ff_kv4_attn_rows(ptr(q), ptr(kpages), ptr(vpages), ptr(block_table), None, None, ptr(ctx_lens), ptr(out), ptr(scratch), batch, nq, hq, hkv, dim,
                              c_longlong(ldq), c_longlong(out.stride(0)), width, blocks, nsplit, c_float(scale), ptr(status_tensor(q.device)), stream_ptr())
    check(rc, "ff_kv4_attn_rows")
    _count(1 if scratch is None else 2)
    return out


def prompt_in_tiles(max_q_len: int, hq: int, hkv: int) -> bool:
    """Whether :func:`attn_prefill_kv4` over so many rows takes the kernel whose keys and values are FP16 tiles in shared memory."""
    return max_q_len * (hq // hkv) > 64


def attn_prefill_kv4(q: torch.Tensor, kpages: torch.Tensor, vpages: torch.Tensor, block_table: torch.Tensor, q_start: torch.Tensor, q_lens: torch.Tensor,
                     ctx_lens: torch.Tensor, max_q_len: int, hq: int, hkv: int, dim: int, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of packed rows over 4-bit pages: sequence b has the ``q_lens[b]`` rows from ``q_start[b]`` on (at most ``max_q_len``), the last of which
    sees ``ctx_lens[b]`` keys. Rows that belong to no sequence stay as they are in ``out`` (undefined without one). Returns ``[rows, hq * dim]``."""
    rows, ldq, blocks = _check_attention("attn_prefill_kv4", q, kpages, vpages, block_table, ctx_lens, hq, hkv, dim, scale, out)
    batch = block_table.shape[0]
    _check_ints("attn_prefill_kv4", batch, q_start, q_lens)
    _check_device("attn_prefill_kv4", q, q_start, q_lens)
    _require(0 < max_q_len, "attn_prefill_kv4: at least one row")
    _require(out is None or not out.is_cuda or (out.data_ptr() % 16 == 0 and out.stride(0) % 8 == 0), "attn_prefill_kv4: output rows aligned to 16 bytes")
    if not q.is_cuda:
        return _attention_ref(q, kpages, vpages, block_table, q_start, q_lens, ctx_lens, hq, hkv, dim, scale, out)
    if out is None:
        out = torch.empty(rows, hq * dim, dtype=BF16, device=q.device)
    if batch == 0 or rows == 0:
        return out
    if prompt_in_tiles(max_q_len, hq, hkv):
        rc = kernels().ff_kv4_attn_tiles(ptr(q), ptr(kpages), ptr(vpages), ptr(block_table), ptr(q_start), ptr(q_lens), ptr(ctx_lens), ptr(out), batch, max_q_len,
                                         hq, hkv, dim, c_longlong(ldq), c_longlong(out.stride(0)), block_table.shape[1], blocks, c_float(scale),
                                         ptr(status_tensor(q.device)), stream_ptr())
        check(rc, "ff_kv4_attn_tiles")
        _count()
        return out
    rc = kernels().ff_kv4_attn_rows(ptr(q), ptr(kpages), ptr(vpages), ptr(block_table), ptr(q_start), ptr(q_lens), ptr(ctx_lens), ptr(out), None, batch, max_q_len,
                                    hq, hkv, dim, c_longlong(ldq), c_longlong(out.stride(0)), block_table.shape[1], blocks, 1, c_float(scale),
                                    ptr(status_tensor(q.device)), stream_ptr())
    check(rc, "ff_kv4_attn_rows")
    _count()
    return out


# ------------------------------------------------------------------------------------------
# copies of pages
# ------------------------------------------------------------------------------------------
def copy_pages(tensors: list[torch.Tensor], src: list[int], dst: list[int]) -> None:
    """In every tensor (first dimension: pages; any type, widths may differ) page ``dst[i]`` becomes a copy of page ``src[i]``, in place. No page is
    written twice, and none that is written is read: those calls are refused. Keys and values of all layers go in one launch."""
    pairs = len(src)
    _require(len(dst) == pairs, "copy_pages: as many sources as destinations")
    _require(len(set(dst)) == pairs and not set(dst) & set(src), "copy_pages: a page that is written is neither read nor written again")
    if pairs == 0 or not tensors:
        return
    first = tensors[0]
    for t in tensors:
        _require(t.dim() > 0 and t.is_contiguous() and t.device == first.device, "copy_pages: contiguous tensors on one device")
        _require(min(min(src), min(dst)) >= 0 and max(max(src), max(dst)) < t.shape[0], "copy_pages: a page outside the cache")
    if not first.is_cuda:
        a, b = torch.tensor(src), torch.tensor(dst)
        for t in tensors:
            t[b] = t[a]
        return
    _check_device("copy_pages", first)
    size = [t[0].numel() * t.element_size() for t in tensors]
    _require(all(n > 0 and n % 16 == 0 and t.data_ptr() % 16 == 0 for n, t in zip(size, tensors)), "copy_pages: pages of whole 16 bytes")
    n = len(tensors)
    base = (ctypes.c_ulonglong * n)(*[t.data_ptr() for t in tensors])
    rc = kernels().ff_copy_pages(base, (c_longlong * n)(*size), n, (ctypes.c_int * pairs)(*src), (ctypes.c_int * pairs)(*dst), pairs, stream_ptr())
    check(rc, "ff_copy_pages")
    _count(-(-n // 160) * -(-pairs // 256))
