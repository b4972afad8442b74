"""A key / value cache that is held in 4 bits, as cases that can be timed and compared: the tokens' keys and values written into its pages
(and read back), the attention of decoded tokens and of prompts over it, and the copies of pages that a forked sequence needs.

A page holds 64 tokens of one head. A group of 32 neighbouring dimensions of a token has codes 0 .. 15 and two BF16 numbers (scale, lo): an
element stands for ``code * scale + lo``, with ``lo`` the group's least element, ``scale`` its span / 15 rounded to BF16 and codes rounded to
the nearest, ties to even. One page is ``64 * D / 2`` bytes of codes, then ``[64 tokens][D / 32][scale, lo]``. Element ``d = 32 j + 8 u + e`` of
a key is nibble ``e // 2 + 4 (e % 2)`` of 32-bit word ``u D / 32 + j`` of the token's row; of a value it is nibble ``e // 2`` of 16-bit unit ``j`` of
the row's chunk ``2 u + e % 2``. Rows of keys are in order. The rows and chunks of values lie such that lanes which read four tokens each meet
no shared-memory bank twice: token k is at row ``k ^ (k // 8 % 2)`` with its chunks ``c`` at ``c ^ 4 (k // 4 % 2)`` where D is 128, and at row
``k ^ (k // 4 % 4)`` where D is 64.

* ``write``: rows of packed queries, keys and values. Queries and keys are turned by a table of cosines and sines (products and their
  sum rounded to BF16, as the framework's rotation rounds them), keys and values go into the pages and are read back.
* ``decode``: ``rows`` query rows of every sequence (1 in a decode step, more where drafts are verified) over ragged contexts.
* ``prompt``: portions of prompts, causal, behind what the cache holds already.
* ``copy``: pages copied to other pages in every layer's key and value tensors.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 64
HEADS = [(32, 8), (64, 8), (64, 4), (32, 32), (28, 4), (8, 1), (24, 8)]
MOST_DECODE = 3 * 131071 * 8 * 128
MOST_PROMPT = 8191 * 8191 * 32 * 128
MOST_ROWS = 8191 * 80 * 128
MOST_COPIED = 64 * 307 * 8 * PAGE * 128 * 2


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def _named(name, case):
    return {"name": name, **case} if name else case


def _write(name, rows, hq, hkv, dim, pad=0, holes=0):
    return _named(name, {"op": "write", "rows": rows, "hq": hq, "hkv": hkv, "dim": dim, "pad": pad, "holes": holes})


def _decode(name, batch, ctx, least, hq, hkv, dim, rows=1, empty=0):
    return _named(name, {"op": "decode", "batch": batch, "ctx": ctx, "least": least, "hq": hq, "hkv": hkv, "dim": dim, "rows": rows, "empty": empty})


def _prompt(name, rows, seqs, past, hq, hkv, dim):
    return _named(name, {"op": "prompt", "rows": rows, "seqs": seqs, "past": past, "hq": hq, "hkv": hkv, "dim": dim})


def _copy(name, layers, blocks, pairs, hkv, dim, held):
    return _named(name, {"op": "copy", "layers": layers, "blocks": blocks, "pairs": pairs, "hkv": hkv, "dim": dim, "held": held})


def listed():
    return [
        # one user's chat: a token's keys and values in the benchmark's model, latency counts
        _write("write 1", 1, 32, 8, 128),
        # a chunk of prompt rows as the scheduler packs it, some of them padding; wide rows
        _write("write 8191", 8191, 64, 8, 128, 8, 90),
        # one user's chat
        _decode("decode 1 x 900", 1, 900, 900, 32, 8, 128),
        # the benchmark's decode batch: 64 requests behind prompts of 1024, three places of the batch unused
        _decode("decode 64 x 1100", 64, 1100, 1030, 32, 8, 128, 1, 3),
        # long documents, few users
        _decode("decode 3 x 131071", 3, 131071, 90000, 64, 8, 128),
        # drafts verified: five rows of every sequence, heads that share their keys 16 to one
        _decode("verify 24 x 4000", 24, 4000, 700, 64, 4, 128, 5),
        # many chats of all lengths over narrow heads
        _decode("decode 200 x 3000 narrow", 200, 3000, 1, 28, 4, 64),
        # a short question
        _prompt("prompt 37", 37, 1, 0, 32, 8, 128),
        # portions of five prompts, some of them far behind their beginnings
        _prompt("prompts 2000 behind 30000", 2000, 5, 30000, 64, 8, 128),
        # a document in one chunk
        _prompt("prompt 8191", 8191, 1, 0, 32, 8, 128),
        # a second sample of a request: its unfinished page in every layer
        _copy("copy 1 page", 32, 257, 1, 8, 128, "4 bits"),
        # a burst of forks of requests over the wide cache
        _copy("copy 150 pages bf16", 32, 307, 150, 8, 128, "bf16"),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["write", "decode", "decode", "decode", "prompt", "prompt", "copy"])
    hq, hkv = rng.choice(HEADS)
    dim = rng.choice([128, 128, 128, 64])
    if op == "write":
        rows = log(1, min(8191, MOST_ROWS // ((hq + 2 * hkv) * dim)))
        return _write(None, rows, hq, hkv, dim, rng.choice([0, 0, 8, 40]), rng.choice([0, 0, rows // 7]))
    if op == "decode":
        rows = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
        batch = log(1, 256)
        ctx = log(rows, max(rows, min(131071, MOST_DECODE // (batch * hkv * dim))))
        return _decode(None, batch, ctx, max(rows, rng.choice([1, ctx // 2, ctx])), hq, hkv, dim, rows, rng.choice([0, 0, batch // 5]))
    if op == "prompt":
        rows = log(1, 8191 if hq <= 32 else 5791)
        room = MOST_PROMPT // (rows * hq * dim)
        past = rng.choice([0, log(1, max(1, min(100000, room - rows)))]) if room > rows else 0
        return _prompt(None, rows, log(1, min(rows, 32)), past, hq, hkv, dim)
    held = rng.choice(["4 bits", "4 bits", "bf16"])
    layers = log(1, 80)
    one = 2 * layers * hkv * (_page_bytes(dim) if held == "4 bits" else PAGE * dim * 2)
    pairs = log(1, max(1, min(150, MOST_COPIED // one // 3)))
    return _copy(None, layers, rng.randint(2 * pairs, max(2 * pairs, min(400, MOST_COPIED // one))), pairs, hkv, dim, held)


def _page_bytes(dim):
    return PAGE * (dim // 2 + dim // 8)


def _lens(case):
    """Keys that the last row of every sequence sees."""
    rng = random.Random(case["ctx"] * 131 + case["batch"])
    live = case["batch"] - case["empty"]
    lens = [case["ctx"]] + [rng.randint(case["least"], case["ctx"]) for _ in range(live - 1)] + [0] * case["empty"]
    rng.shuffle(lens)
    return lens


def _spans(case):
    """(rows, keys in front of them) of every sequence of a prompt case."""
    rng = random.Random(case["rows"] * 17 + case["seqs"])
    cuts = sorted(rng.sample(range(1, case["rows"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
    takes = [b - a for a, b in zip([0] + cuts, cuts + [case["rows"]])]
    pasts = [case["past"]] + [rng.choice([0, rng.randint(0, case["past"])]) for _ in range(case["seqs"] - 1)]
    return list(zip(takes, pasts))


def work(case):
    hkv, dim = case["hkv"], case["dim"]
    page = _page_bytes(dim)
    if case["op"] == "copy":
        one = page if case["held"] == "4 bits" else PAGE * dim * 2
        return {"bytes": 2 * 2 * case["layers"] * case["pairs"] * hkv * one, "flops": 0}
    hq = case["hq"]
    if case["op"] == "write":
        # rows in, queries out; pages out and in again, values out
        return {"bytes": case["rows"] * (2 * (2 * hq + 4 * hkv) * dim + 4 * hkv * page // PAGE + 4 * dim), "flops": 0}
    if case["op"] == "decode":
        lens, n = _lens(case), case["rows"]
        pairs = sum(n * c - n * (n - 1) // 2 for c in lens if c)
        rows = n * case["batch"]
    else:
        spans = _spans(case)
        lens, rows = [t + p for t, p in spans], case["rows"]
        pairs = sum(t * p + t * (t + 1) // 2 for t, p in spans)
    return {"bytes": 2 * hkv * page * sum(lens) // PAGE + 2 * 2 * rows * hq * dim, "flops": 4.0 * dim * hq * pairs}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _random_pages(blocks, hkv, dim, gen, spread):
    """Pages as a cache holds them after keys or values with outlying channels: codes thick in the middle, spans of all sizes."""
    groups = dim // 32
    pages = torch.empty(blocks, hkv, _page_bytes(dim), dtype=torch.uint8, device="cuda")
    for at in range(0, blocks, 256):
        part = pages[at: at + 256]
        n = part.shape[0]
        nib = torch.randn(2, n, hkv, PAGE * dim // 2, generator=gen, device="cuda", dtype=torch.float16).mul_(3.3).add_(7.5).round_().clamp_(0, 15).to(torch.uint8)
        part[:, :, : PAGE * dim // 2] = nib[0] | (nib[1] << 4)
        span = torch.exp(torch.randn(n, hkv, PAGE, groups, generator=gen, device="cuda") * 0.4) * spread
        mid = torch.randn(n, hkv, PAGE, groups, generator=gen, device="cuda") * 0.2 * spread
        stats = torch.stack([span / 15, mid - span / 2], dim=-1).to(torch.bfloat16)
        part[:, :, PAGE * dim // 2:] = stats.flatten(2).view(torch.uint8)
    return pages


def _table(lens, gen, width):
    """Pages of every sequence in any order, and how many there are."""
    need = [-(-c // PAGE) for c in lens]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(len(lens), max(width, 1), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at: at + n]
        at += n
    return blocks, table.cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    hkv, dim = case["hkv"], case["dim"]
    state = {k: case[k] for k in ("op", "hkv", "dim")}
    if case["op"] == "copy":
        shape, blocks = (hkv, _page_bytes(dim)) if case["held"] == "4 bits" else (hkv, PAGE, dim), case["blocks"]
        make = lambda: torch.randint(256, (blocks, *shape), generator=gen, device="cuda", dtype=torch.uint8) if len(shape) == 2 else normal(blocks, *shape).to(torch.bfloat16)
        ids = random.Random(seed).sample(range(blocks), 2 * case["pairs"])
        return {**state, "tensors": [make() for _ in range(2 * case["layers"])], "src": ids[: case["pairs"]], "dst": ids[case["pairs"]:]}
    hq = case["hq"]
    state.update(hq=hq, scale=1 / math.sqrt(dim))
    if case["op"] == "write":
        rows, width = case["rows"], (hq + 2 * hkv) * dim
        gain = torch.exp(normal(1, width) * 0.5)                      # channels differ, some stand out
        qkv = torch.zeros(rows, width + case["pad"], device="cuda", dtype=torch.bfloat16)
        qkv[:, :width] = (normal(rows, width) * gain + 0.5 * normal(1, width)).to(torch.bfloat16)
        first = random.Random(seed).randint(0, 100000)
        angle = (torch.arange(rows, device="cuda", dtype=torch.float64) + first)[:, None] / 500000.0 ** (torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        turn = torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1).to(torch.bfloat16).float().contiguous()
        blocks = -(-rows // PAGE) + 2
        slots = torch.randperm(blocks, generator=gen, device="cuda")[:, None] * PAGE + torch.arange(PAGE, device="cuda")
        slots = slots.flatten()[5: 5 + rows].to(torch.int32).contiguous()                  # the first page begins inside
        if case["holes"]:
            slots[torch.randperm(rows, generator=gen, device="cuda")[: case["holes"]]] = -1
        pages = [torch.zeros(blocks, hkv, _page_bytes(dim), dtype=torch.uint8, device="cuda") for _ in range(2)]
        return {**state, "qkv": qkv[:, :width], "turn": turn, "slots": slots, "kpages": pages[0], "vpages": pages[1]}
    if case["op"] == "decode":
        lens, rows, n = _lens(case), case["rows"] * case["batch"], case["rows"]
        takes = [n] * case["batch"]
        state["nq"] = n
    else:
        takes, pasts = zip(*_spans(case))
        lens, rows = [t + p for t, p in zip(takes, pasts)], case["rows"]
        starts = np.concatenate([[0], np.cumsum(takes)[:-1]])
        state.update(q_start=torch.tensor(starts, dtype=torch.int32).cuda(), q_lens=torch.tensor(takes, dtype=torch.int32).cuda(), most=max(takes))
    blocks, table = _table(lens, gen, -(-max(lens) // PAGE))
    # the queries are the first columns of packed rows, as the projection leaves them
    q = normal(rows, (hq + 2 * hkv) * dim).to(torch.bfloat16)[:, : hq * dim]
    return {**state, "q": q, "kpages": _random_pages(blocks, hkv, dim, gen, 4.0), "vpages": _random_pages(blocks, hkv, dim, gen, 2.0), "table": table,
            "ctx": torch.tensor(lens, dtype=torch.int32).cuda(), "spans": list(zip(takes, lens))}


# ------------------------------------------------------------------------------------------
# the operators
# ------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from flyingfish_b200.ops import kv4_ops
        if s["op"] == "copy":
            kv4_ops.copy_pages(s["tensors"], s["src"], s["dst"])
            return s["tensors"]
        if s["op"] == "write":
            q = kv4_ops.write_kv4(s["qkv"], s["slots"], s["kpages"], s["vpages"], s["hq"], s["hkv"], s["dim"], cos_sin=s["turn"])
            return (q, *kv4_ops.read_kv4(s["kpages"], s["vpages"], s["slots"], s["dim"]))
        args = (s["q"], s["kpages"], s["vpages"], s["table"])
        if s["op"] == "decode":
            return kv4_ops.attn_decode_kv4(*args, s["ctx"], s["hq"], s["hkv"], s["dim"], s["scale"], nq=s["nq"])
        return kv4_ops.attn_prefill_kv4(*args, s["q_start"], s["q_lens"], s["ctx"], s["most"], s["hq"], s["hkv"], s["dim"], s["scale"])
    if s["op"] == "copy":
        src, dst = (torch.tensor(v, device=s["tensors"][0].device) for v in (s["src"], s["dst"]))
        for t in s["tensors"]:
            t[dst] = t[src]
        return s["tensors"]
    if s["op"] == "write":
        return _plain_write(s)
    return _plain_attention(s)


def _bf16_of_double(x):
    """One rounding to BF16 (a cast goes through 32 bits)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256) / 256, e)


def _plain_write(s):
    hq, hkv, dim = s["hq"], s["hkv"], s["dim"]
    rows = s["qkv"].shape[0]
    x = s["qkv"].float().view(rows, hq + 2 * hkv, dim)
    r16 = lambda t: t.to(torch.bfloat16).float()
    c, sn = s["turn"][:, None, :, 0], s["turn"][:, None, :, 1]
    a, b = x[:, : hq + hkv, : dim // 2], x[:, : hq + hkv, dim // 2:]
    turned = torch.cat([r16(r16(a * c) - r16(b * sn)), r16(r16(b * c) + r16(a * sn))], dim=-1)
    out = []
    for part in (turned[:, hq:], x[:, hq + hkv:]):
        g = part.double().view(rows, hkv, dim // 32, 32)              # next to the codes' borders 32 bits would not do
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        scale = _bf16_of_double((hi - lo) / 15)
        scale = torch.where(scale < 2.0 ** -126, 0.0, scale)
        code = torch.where(scale > 0, torch.round((g - lo) / torch.where(scale > 0, scale, 1.0)).clamp(0, 15), 0.0)
        value = (code * scale + lo).view(rows, hkv, dim)
        out.append(torch.where(s["slots"][:, None, None] >= 0, value, 0.0).to(torch.bfloat16))
    return turned[:, :hq].reshape(rows, hq * dim).to(torch.bfloat16), *out


def _plain_values(pages, dim, of_keys):
    """What pages [n, heads, bytes] stand for, as FP32 [heads, n * 64, dim]."""
    n, heads, _ = pages.shape
    groups = dim // 32
    codes, stats = pages[..., : PAGE * dim // 2], pages[..., PAGE * dim // 2:]
    stats = stats.contiguous().view(torch.bfloat16).view(n, heads, PAGE, groups, 1, 2).float()
    nib = torch.stack([codes & 15, codes >> 4], dim=-1).view(n, heads, PAGE, dim)
    if of_keys:
        # [u][j][odd][half of e] -> [j][u][half of e][odd]
        code = nib.view(n, heads, PAGE, 4, groups, 2, 4).permute(0, 1, 2, 4, 3, 6, 5)
    else:
        k = torch.arange(PAGE, device=pages.device)
        chunk = torch.arange(8, device=pages.device)
        if dim == 128:
            row, at = k ^ (k // 8 % 2), chunk[None, :] ^ (4 * (k // 4 % 2))[:, None]
        else:
            row, at = k ^ (k // 4 % 4), chunk[None, :].expand(PAGE, 8)
        code = nib.view(n, heads, PAGE, 8, groups, 4)[:, :, row[:, None], at]
        # [u][odd][j][half of e] -> [j][u][half of e][odd]
        code = code.view(n, heads, PAGE, 4, 2, groups, 4).permute(0, 1, 2, 5, 3, 6, 4)
    value = code.reshape(n, heads, PAGE, groups, 32).float() * stats[..., 0] + stats[..., 1]
    return value.view(n, heads, PAGE, dim).transpose(0, 1).reshape(heads, n * PAGE, dim)


def _plain_attention(s):
    hq, hkv, dim = s["hq"], s["hkv"], s["dim"]
    share = hq // hkv
    outs, row = [], 0
    for i, (take, ctx) in enumerate(s["spans"]):
        q = s["q"][row: row + take].float().view(take, hkv, share, dim).permute(1, 2, 0, 3)
        row += take
        if ctx == 0:
            outs.append(torch.zeros(take, hq * dim, device=q.device, dtype=torch.bfloat16))
            continue
        pages = s["table"][i, : -(-ctx // PAGE)].long()
        keys = _plain_values(s["kpages"][pages], dim, True)[:, :ctx]
        values = _plain_values(s["vpages"][pages], dim, False)[:, :ctx]
        out = torch.empty(hkv, share, take, dim, device=q.device)
        upto = torch.arange(ctx, device=q.device)[None, :] <= torch.arange(ctx - take, ctx, device=q.device)[:, None]
        for h in range(hkv):
            score = (q[h].reshape(share * take, dim) @ keys[h].T).view(share, take, ctx) * s["scale"]
            score = score.masked_fill_(~upto, float("-inf"))
            p = score.sub_(score.amax(-1, keepdim=True)).exp_()
            out[h] = (p.view(share * take, ctx) @ values[h]).view(share, take, dim) / p.sum(-1, keepdim=True)
        outs.append(out.permute(2, 0, 1, 3).reshape(take, hq * dim).to(torch.bfloat16))
    return torch.cat(outs)


# ------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        # nothing is computed: which page lies where
        where = torch.arange(case["blocks"])
        for a, b in zip(s["src"], s["dst"]):
            where[b] = a
        return [t.index_select(0, where.to(t.device)) for t in s["tensors"]]
    if case["op"] == "write":
        return _exact_write(s)
    return _exact_attention(s)


def _exact_write(s):
    hq, hkv, dim = s["hq"], s["hkv"], s["dim"]
    x = s["qkv"].double().reshape(-1, hq + 2 * hkv, dim)
    cos, sin = (torch.cat([s["turn"][:, :, i].double()] * 2, dim=1)[:, None] for i in (0, 1))
    narrow = lambda a: a.to(torch.float32).to(torch.bfloat16).double()           # the rotation's roundings are part of what it is
    head = x[:, : hq + hkv]
    other = torch.cat([-head[..., dim // 2:], head[..., : dim // 2]], dim=-1)
    head = narrow(narrow(head * cos) + narrow(other * sin))
    live = (s["slots"] >= 0)[:, None, None]
    values = []
    for part in (head[:, hq:], x[:, hq + hkv:]):
        out = torch.zeros_like(part)
        for j in range(0, dim, 32):
            g = part[..., j: j + 32]
            lo = g.min(-1, keepdim=True).values
            step = ((g.max(-1, keepdim=True).values - lo) / 15).cpu().numpy()
            mant, expo = np.frexp(step)
            step = np.ldexp(np.rint(np.ldexp(mant, 8)), expo - 8)                  # eight bits, ties to even
            step = torch.from_numpy(np.where(step < 2.0 ** -126, 0.0, step)).to(g.device)
            out[..., j: j + 32] = torch.nan_to_num(torch.round((g - lo) / step), nan=0.0).clamp(0, 15) * step + lo
        values.append(torch.where(live, out, 0.0))
    return head[:, :hq].reshape(len(x), hq * dim), *values


def _places(dim, of_keys):
    """Byte and shift of every (token, element) of a page's codes."""
    k, d = torch.meshgrid(torch.arange(PAGE), torch.arange(dim), indexing="ij")
    j, u, e = d // 32, d % 32 // 8, d % 8
    if of_keys:
        nibble = e // 2 + 4 * (e % 2)
        byte = k * (dim // 2) + 4 * (u * (dim // 32) + j) + nibble // 2
    else:
        nibble, lane = e // 2, 2 * u + e % 2
        row = torch.where(k & 8 > 0, k ^ 1, k) if dim == 128 else k - k % 4 + (k % 4 ^ k // 4 % 4)
        if dim == 128:
            lane = torch.where(k & 4 > 0, lane ^ 4, lane)
        byte = row * (dim // 2) + lane * (dim // 16) + 2 * j + nibble // 2
    return byte, 4 * (nibble % 2)


def _exact_values(pages, dim, of_keys):
    byte, shift = (t.to(pages.device) for t in _places(dim, of_keys))
    code = (pages[:, byte] >> shift.to(torch.uint8)) & 15
    stats = pages[:, PAGE * dim // 2:].contiguous().view(torch.bfloat16).double().view(-1, PAGE, dim // 32, 2).repeat_interleave(32, dim=2)
    return (code.double() * stats[..., 0] + stats[..., 1]).flatten(0, 1)


def _exact_attention(s):
    hq, hkv, dim = s["hq"], s["hkv"], s["dim"]
    out = torch.zeros(s["q"].shape[0], hq, dim, dtype=torch.float64, device="cuda")
    row = 0
    for i, (take, ctx) in enumerate(s["spans"]):
        if ctx:
            pages = s["table"][i, : -(-ctx // PAGE)].long()
            first = torch.arange(ctx - take, ctx, device="cuda")
            for kv in range(hkv):
                keys, values = _exact_values(s["kpages"][pages, kv], dim, True)[:ctx], _exact_values(s["vpages"][pages, kv], dim, False)[:ctx]
                for h in range(kv * (hq // hkv), (kv + 1) * (hq // hkv)):
                    q = s["q"][row: row + take, h * dim: (h + 1) * dim].double()
                    for at in range(0, take, 1024):
                        logit = torch.einsum("rd,kd->rk", q[at: at + 1024], keys) * s["scale"]
                        logit[torch.arange(ctx, device="cuda")[None, :] > first[at: at + 1024, None]] = -math.inf
                        out[row + at: row + min(at + 1024, take), h] = torch.softmax(logit, dim=1) @ values
        row += take
    return out.view(-1, hq * dim)
