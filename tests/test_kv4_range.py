"""Attention over 4-bit pages whose values (and keys) are of any size that a page holds, against the pages' values in 64 bits.

Bounds are relative to the terms themselves, so they shrink with the values. With p the weights, v the values, lo a group's least element and M(k) the greatest
magnitude of a scale or lo in key k's page:
* the result's rounding to BF16, half a step: 2^-8 of it;
* few rows: p scale, p and lo rounded to FP16, 2^-11 each: of p (v - lo), and twice of p |lo|, which is at most p (v - lo) + p |v|;
* prompts in tiles: p and v rounded to FP16, 2^-11 of p |v| each, of keys that are rounded to 11 bits;
* FP32 arithmetic (sums in other orders, exponentials of FP32 scores): 2^-14 of p |v| and of p (v - lo);
* what is too small for FP16 beside the greatest of its page, M(k). Few rows: p, lo and p scale are held to 2^-25 where p is multiplied by 2^7, scale and lo by 2^7 over a
  power of two that is at most 2^5 M(k) (the power of an earlier page is kept while it is less than five binades above this one's): a weight is off by 2^-32 beside the greatest weight, times |lo|, a lo
  by 2^-32 x 2^5 M(k), times p, and a product p scale by 2^-39 x 2^5 M(k), times a code of 15. Together less than 2^-27 M(k) (p + 2^-3 of the greatest weight);
* in tiles p is multiplied by 2^7 and the values by 2^13 over a power of two that is at most 2^11 M(k) (16 scale counts there, a binade is to spare, seven are kept): a scale or lo off by
  2^-25 makes an element of code 15 off by less than 2^-20, that is 2^-22 M(k), times p; a weight is off by 2^-32 of the greatest, times |v|, at most 16 M(k);
* a power of two is kept within 2^60 of the greatest so far, which no page here needs."""
import math

import pytest
import torch

from flyingfish_b200 import ops
from flyingfish_b200.ops import kv4_ops
from flyingfish_b200.ops.kv4_ops import PAGE
from test_kv4 import _cache, _rows

BF16 = torch.bfloat16
E = 2.0 ** -8


def _resize(pages, dim, power, block=None, tokens=slice(None)):
    """What the pages' elements stand for, times 2^power: exact (unwritten places hold no numbers and stay so)."""
    stats = pages[..., PAGE * dim // 2:].contiguous().view(BF16).unflatten(-1, (PAGE, dim // 32 * 2))
    at = slice(None) if block is None else block
    part = stats[at][..., tokens, :]
    stats[at, :, tokens] = torch.where(part.isfinite(), torch.ldexp(part.float(), torch.tensor(power, device=part.device)).to(BF16), part)
    pages[..., PAGE * dim // 2:] = stats.flatten(-2).view(torch.uint8)


def _terms(q, kpages, vpages, table, spans, hq, hkv, dim, scale, key_bits):
    """Per row and head: the attention in 64 bits, sums of p |v| and of p (v - lo), and of M(k) (p + 2^-3 of the greatest p). ``key_bits``: keys rounded to so many bits first."""
    g = hq // hkv
    res, mag, off, small = (torch.zeros(q.shape[0], hq, dim, dtype=torch.float64) for _ in range(4))
    for b, (at, n, ctx) in enumerate(spans):
        if ctx <= 0 or n == 0:
            continue
        pages = table[b, : -(-ctx // PAGE)].long().cpu()
        k, v = (kv4_ops.page_values(p.cpu()[pages], dim, keys).double().transpose(0, 1).reshape(hkv, -1, dim)[:, :ctx] for p, keys in ((kpages, True), (vpages, False)))
        stats = vpages.cpu()[pages][..., PAGE * dim // 2:].contiguous().view(BF16).double().unflatten(-1, (PAGE, dim // 32, 2)).transpose(0, 1).reshape(hkv, -1, dim // 32, 2)[:, :ctx]
        lo = stats[..., 1].repeat_interleave(32, -1)
        most = stats.abs().flatten(2).amax(-1)
        most = torch.nn.functional.pad(most, (0, -ctx % PAGE)).unflatten(-1, (-1, PAGE)).amax(-1, keepdim=True).expand(-1, -1, PAGE).flatten(1)[:, :ctx]
        if key_bits is not None:
            m, e = torch.frexp(k)
            k = torch.ldexp(torch.round(m * 2 ** key_bits) / 2 ** key_bits, e)
        x = q[at: at + n, : hq * dim].double().cpu().view(n, hkv, g, dim)
        score = torch.einsum("nhgd,hkd->nhgk", x, k) * scale
        score.masked_fill_((torch.arange(ctx)[None, :] > torch.arange(ctx - n, ctx)[:, None])[:, None, None], -math.inf)
        p = torch.softmax(score, dim=-1)
        each = lambda w, t: torch.einsum("nhgk,hkd->nhgd", w, t).reshape(n, hq, dim)
        res[at: at + n], mag[at: at + n], off[at: at + n] = each(p, v), each(p, v.abs()), each(p, v - lo)
        small[at: at + n] = torch.einsum("nhgk,hk->nhg", p + 0.125 * p.amax(-1, keepdim=True), most).reshape(n, hq, 1)
    return [t.view(q.shape[0], hq * dim) for t in (res, mag, off, small)]


def _check(got, res, mag, off, small, tiles):
    tol = res.abs() * E + (2 * mag if tiles else 2 * off + 2 * mag) * 2.0 ** -11 + (mag + off) * 2.0 ** -14 + small * (2.0 ** -22 if tiles else 2.0 ** -27)
    err = (got.cpu().double() - res).abs()
    worst = float((err / tol.clamp_min(1e-300)).max())
    assert worst <= 1, f"{worst} of the tolerance; off by {float(err.norm() / res.norm())} of the result"


def _run(q, kp, vp, table, lens, hq, hkv, dim, scale, nq=1):
    tiles = kv4_ops.in_tiles(nq, hq, hkv)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = kv4_ops.attn_decode_kv4(q, kp, vp, table, ctx, hq, hkv, dim, scale, nq=nq)
    assert ops.read_status()[0] == 0
    # keys of a tile are FP16 numbers: 11 bits
    _check(got, *_terms(q, kp, vp, table, [(i * nq, nq, c) for i, c in enumerate(lens)], hq, hkv, dim, scale, 11 if tiles else None), tiles)


FEW = [(128, 8, 2, 1, [900, 70]), (64, 7, 1, 3, [2000, 3]), (128, 16, 1, 2, [5000]), (64, 4, 4, 1, [20000])]
MANY = [(128, 16, 1, 9, [300, 2500]), (64, 4, 4, 70, [700]), (128, 8, 2, 40, [1500, 64, 5000]), (64, 28, 4, 9, [64, 12000])]


def _dominant(q, kp, vp, table, hq, hkv, dim, scale, nq, blocks, nats):
    """The first key of every sequence ``nats`` above the others, whose scores are next to nothing."""
    for b, block in enumerate(blocks):
        k = kv4_ops.page_values(kp[block][None].cpu(), dim, True)[0, :, 0]                       # [hkv, dim]
        want = (k * (nats / scale) / k.square().sum(-1, keepdim=True)).repeat_interleave(hq // hkv, 0)
        q[b * nq: (b + 1) * nq, : hq * dim] = want.flatten().to(BF16).to(q.device)


def _made(dim, hq, hkv, nq, lens, seed=3):
    kp, vp, table = _cache(lens, hkv, dim, seed, "cuda", width=-(-max(lens) // PAGE) + 1)
    q = _rows(len(lens) * nq, (hq + 2 * hkv) * dim, 11).cuda()
    return kp, vp, table, q, 1 / math.sqrt(dim)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [7, 0, -10, -14, -20, -40, -100])
@pytest.mark.parametrize("dim,hq,hkv,nq,lens", FEW + MANY)
def test_values_of_any_size(dim, hq, hkv, nq, lens, power):
    kp, vp, table, q, scale = _made(dim, hq, hkv, nq, lens)
    _resize(vp, dim, power)
    _run(q, kp, vp, table, lens, hq, hkv, dim, scale, nq)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [0, -10, -14, -20])
@pytest.mark.parametrize("nats", [8, 13])
@pytest.mark.parametrize("dim,hq,hkv,nq,lens", FEW + MANY)
def test_a_key_far_above_the_others(dim, hq, hkv, nq, lens, nats, power):
    kp, vp, table, q, scale = _made(dim, hq, hkv, nq, lens)
    first = [int(table[i, 0]) for i in range(len(lens))]
    _dominant(q, kp, vp, table, hq, hkv, dim, scale, nq, first, nats)
    _resize(kp, dim, -8)
    for b in first:
        _resize(kp, dim, 8, b, slice(0, 1))
    _resize(vp, dim, power)
    for b in first[:1]:                                             # the key that has the weight has values next to nothing, as first tokens do
        _resize(vp, dim, -9, b, slice(0, 1))
    _run(q, kp, vp, table, lens, hq, hkv, dim, scale, nq)


@pytest.mark.gpu
@pytest.mark.parametrize("powers", [(0, 7, -8, 3), (-20, 4, -3, -30), (-30, -6, 0, 7), (7, -2, -12, -30)])
@pytest.mark.parametrize("dim,hq,hkv,nq,lens", FEW + MANY)
def test_pages_whose_values_differ(dim, hq, hkv, nq, lens, powers):
    kp, vp, table, q, scale = _made(dim, hq, hkv, nq, lens)
    for i, c in enumerate(lens):
        for p in range(-(-c // PAGE)):
            _resize(vp, dim, powers[p % len(powers)], int(table[i, p]))
            if p % 7 == 5:                                          # a page of zeros
                vp[int(table[i, p])] = 0
    _run(q, kp, vp, table, lens, hq, hkv, dim, scale, nq)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [7, -10, -20, -60])
@pytest.mark.parametrize("dim,hq,hkv,nq,lens", FEW + MANY)
def test_keys_of_any_size(dim, hq, hkv, nq, lens, power):
    """Queries that make up for it; pages of keys differ by 2^6."""
    kp, vp, table, q, scale = _made(dim, hq, hkv, nq, lens)
    q.copy_(torch.ldexp(q.float(), torch.tensor(-power, device="cuda")).to(BF16))
    _resize(kp, dim, power)
    for i, c in enumerate(lens):
        for p in range(1, -(-c // PAGE), 3):
            _resize(kp, dim, -6, int(table[i, p]))
    _run(q, kp, vp, table, lens, hq, hkv, dim, scale, nq)


def test_lanes_that_wait_give_up_together():
    """In the kernel of few rows every warp waits as a whole: each wait that may run out is voted on, or lanes that go on would wait for those that gave up."""
    from pathlib import Path
    source = (Path(kv4_ops.__file__).parent / "csrc" / "attention_kv4.cu").read_text()
    assert source.count("mbar_wait(") == source.count("__all_sync(0xffffffffu, mbar_wait(") == 2
