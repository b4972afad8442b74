"""What a request of a shared batch brings along of its own, as cases that can be timed and compared: the low-rank adapter that is
added to a projection for its rows, and the settings with which its next token is drawn.

* ``lora``: ``y = x W^T`` plus, for every row with an adapter, ``scale (x A^T) B^T`` of that adapter. Weights are BF16 in the layouts that
  the framework's projections and its adapter stacks have; the adapters of a stack have different ranks and are padded with zeros.
* ``sample``: temperature, top-k, top-p and min-p of every row, from a given random number per row.

A ``lora`` case has ``requests`` requests that share ``rows`` rows (one each in a decode step, a portion of a prompt otherwise); ``bare`` of them
have no adapter, the others use ``used`` of the ``adapters`` that are resident.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
MODES = ("mixed", "top_p", "top_k", "min_p", "all", "plain")
MOST_WORK = 8191 * 4096 * 14336


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------
def _lora(name, rows, requests, bare, used, adapters, k, n, rank):
    c = {"op": "lora", "rows": rows, "requests": requests, "bare": bare, "used": used, "adapters": adapters, "k": k, "n": n, "rank": rank}
    return {"name": name, **c} if name else c


def _sample(name, rows, vocab, dtype, mode, sigma, pad=0):
    c = {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mode": mode, "sigma": sigma, "pad": pad}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user's chat with a fine-tuned adapter: a token's output projection, latency counts
        _lora("lora decode 1", 1, 1, 0, 1, 8, 4096, 4096, 16),
        # a few users, some with the base model; the down projection
        _lora("lora decode 7 down", 7, 7, 2, 3, 16, 14336, 4096, 32),
        # a full decode batch in which everyone has an adapter of their own; the fused QKV projection
        _lora("lora decode 64 qkv", 64, 64, 0, 64, 64, 4096, 6144, 16),
        # one popular adapter, with half of the requests on it; the widest projection
        _lora("lora decode 113 wide", 113, 113, 56, 1, 4, 4096, 28672, 64),
        # a burst of short prompts under different adapters, a row count that fills no tile
        _lora("lora prompts 300", 300, 9, 2, 5, 16, 4096, 6144, 16),
        # a document with one adapter
        _lora("lora prompt 1000", 1000, 1, 0, 1, 8, 4096, 4096, 64),
        # a chunk of prompt rows as the scheduler packs it; the down projection
        _lora("lora prompts 8191 down", 8191, 12, 3, 6, 16, 14336, 4096, 16),
        # one user's chat: nucleus sampling over the vocabulary of the benchmark's model
        _sample("sample 1", 1, 128256, "bf16", "top_p", 2.5),
        # a decode batch with every user's own settings, greedy ones among them
        _sample("sample 64 mixed", 64, 128256, "bf16", "mixed", 2.5),
        # 32-bit logits of a vocabulary that fills no vector, in rows of a wider buffer; flat distributions, top-k only
        _sample("sample 33 top-k fp32", 33, 50257, "fp32", "top_k", 1.0, 7),
        # the whole distribution, no filter: what evaluation by sampling does
        _sample("sample 48 plain fp32", 48, 129280, "fp32", "plain", 1.5),
        # the largest decode batch and the largest vocabulary
        _sample("sample 256 all", 256, 151936, "bf16", "all", 2.5),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        rows = log(1, 256)
        vocab = min(log(1000, 262144), 256 * 151936 // rows)
        return _sample(None, rows, vocab, rng.choice(["bf16", "bf16", "fp32"]), rng.choice(MODES), round(rng.uniform(0.5, 3.0), 2), rng.choice([0, 0, 1, 8, 24]))
    k, n = (8 * log(32, 1792) if rng.random() < 0.5 else rng.choice([1024, 2048, 4096, 6144, 8192, 14336]) for _ in range(2))
    rows = log(1, 128) if rng.random() < 0.5 else log(129, max(129, min(8191, MOST_WORK // (k * n))))
    requests = rows if rows <= 128 and rng.random() < 0.8 else log(1, min(rows, 64))
    adapters = log(1, 64)
    bare = rng.choice([0, 0, requests // 3, rng.randint(0, requests)])
    used = rng.randint(1, min(adapters, requests - bare)) if requests > bare else 0
    return _lora(None, rows, requests, bare, used, adapters, k, n, rng.choice([16, 16, 32, 48, 64, 128]))


def _ranks(case):
    """Ranks of the adapters in use: every other one has half the stack's width."""
    return [case["rank"] // (1 + j % 2) for j in range(case["used"])]


def work(case):
    if case["op"] == "sample":
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["rows"] * (case["vocab"] * size + 5 * 4 + 8), "flops": 0}
    m, k, n = case["rows"], case["k"], case["n"]
    ranks = sum(_ranks(case))
    share = 1.0 - case["bare"] / case["requests"]
    mean = ranks / case["used"] if case["used"] else 0.0
    return {"bytes": 2 * (m * k + n * k + m * n + ranks * (k + n)) + 4 * m, "flops": 2.0 * m * n * k + 2.0 * m * share * mean * (k + n)}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    if case["op"] == "sample":
        return _prepare_sample(case, seed, gen, normal)
    rng = random.Random(seed)
    m, k, n, r, count = case["rows"], case["k"], case["n"], case["rank"], case["adapters"]
    # the requests' adapters: every one of those in use at least once, in any order
    which = rng.sample(range(count), case["used"])
    mine = [which[i % case["used"]] for i in range(case["requests"] - case["bare"])] + [-1] * case["bare"]
    rng.shuffle(mine)
    cuts = sorted(rng.sample(range(1, m), case["requests"] - 1)) if case["requests"] > 1 else []
    ids = torch.repeat_interleave(torch.tensor(mine, dtype=torch.int32), torch.tensor([b - a for a, b in zip([0] + cuts, cuts + [m])]))
    ranks = torch.full((count,), r, dtype=torch.int32)
    ranks[torch.tensor(which, dtype=torch.long)] = torch.tensor(_ranks(case), dtype=torch.int32)
    ranks = ranks.cuda()
    live = torch.arange(r, device="cuda")[None, :] < ranks[:, None]                    # ranks behind an adapter's own are zero
    a = (normal(count, r, k) / math.sqrt(k) * live[:, :, None]).to(torch.bfloat16)
    b = (normal(count, n, r) * 0.02 * live[:, None, :]).to(torch.bfloat16)
    return {"op": "lora", "x": normal(m, k).to(torch.bfloat16), "w": (normal(n, k) * 0.02).to(torch.bfloat16), "a": a, "b": b,
            "scale": torch.full((count,), 2.0, device="cuda") / (1 + torch.arange(count, device="cuda") % 3), "ranks": ranks, "ids": ids.cuda()}


def _prepare_sample(case, seed, gen, normal):
    rows, vocab = case["rows"], case["vocab"]
    # a broad bulk and some tokens that fit: what a language model's head gives
    logits = normal(rows, vocab) * case["sigma"]
    few = torch.randint(vocab, (rows, 48), generator=gen, device="cuda")
    lift = torch.rand(rows, 48, generator=gen, device="cuda") * 6.0 * case["sigma"]
    logits = logits.scatter_add_(1, few, lift).to(DTYPES[case["dtype"]])
    wide = torch.full((rows, vocab + case["pad"]), 1e4, dtype=logits.dtype, device="cuda")
    wide[:, :vocab] = logits
    rng, mode = random.Random(seed), case["mode"]
    settings = []
    for _ in range(rows):
        kind = rng.choice(["greedy", "top_p", "top_k", "min_p", "all", "plain"]) if mode == "mixed" else mode
        settings.append((0.0 if kind == "greedy" else round(rng.uniform(0.6, 1.3), 2), rng.choice([1, 20, 50, 200]) if kind in ("top_k", "all") else 0,
                         round(rng.uniform(0.8, 0.99), 2) if kind in ("top_p", "all") else 1.0,
                         round(rng.uniform(0.01, 0.2), 3) if kind in ("min_p", "all") else 0.0))
    t, top_k, top_p, min_p = zip(*settings)
    column = lambda v, dtype=torch.float32: torch.tensor(v, dtype=dtype, device="cuda")
    return {"op": "sample", "logits": wide[:, :vocab], "uniforms": torch.rand(rows, generator=gen, device="cuda"), "temperature": column(t),
            "top_k": column(top_k, torch.int32), "top_p": column(top_p), "min_p": column(min_p)}


# ------------------------------------------------------------------------------------------
# the operators
# ------------------------------------------------------------------------------------------
def run(state):
    if state["op"] == "sample":
        args = [state[k] for k in ("logits", "uniforms", "temperature", "top_k", "top_p", "min_p")]
        if own:
            from flyingfish_b200.ops import sample_ops
            return sample_ops.sample_tokens(*args)
        return _plain_sample(*args)
    if own:
        from flyingfish_b200.ops import lora_ops
        stack = lora_ops.AdapterStack(state["a"], state["b"], state["scale"], state["ranks"])
        return lora_ops.linear_lora(state["x"], state["w"], stack, state["ids"])
    return _plain_lora(*(state[k] for k in ("x", "w", "a", "b", "scale", "ids")))


def _plain_lora(x, w, a, b, scale, ids):
    """All adapters of the stack for all rows, with the factor zero where a row has another adapter or none."""
    x = x.float()
    t = (x @ a.float().flatten(0, 1).T).view(x.shape[0], *a.shape[:2])
    factor = scale * (ids[:, None] == torch.arange(a.shape[0], device=ids.device))
    t = (t * factor[:, :, None]).flatten(1)
    return (x @ w.float().T + t @ b.float().transpose(1, 2).flatten(0, 1)).to(torch.bfloat16)


def _plain_sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """In 64 bits: sums over a vocabulary next to the number that is looked for."""
    vocab = logits.shape[1]
    greedy = temperature == 0
    heat = torch.where(greedy, 1.0, temperature).double()
    top, order = torch.sort(logits, dim=1, descending=True, stable=True)
    away = (top.double() - top[:, :1].double()) / heat[:, None]
    mass = torch.exp(away)
    before = torch.cumsum(mass, 1) - mass                                 # mass of the tokens in front of each
    limit = top_p.double() * mass.sum(1)
    rank = torch.arange(vocab, device=logits.device)
    kept = ((top_k[:, None] <= 0) | (rank < top_k[:, None])) & ((top_p[:, None] >= 1) | (before < limit[:, None]) | (rank == 0))
    kept &= (min_p[:, None] <= 0) | (away >= torch.log(min_p.double())[:, None])
    kept &= ~greedy[:, None] | (rank == 0)
    mass = torch.zeros_like(mass).scatter_(1, order, torch.where(kept, mass, 0.0))       # back in the order of the ids
    upto = torch.cumsum(mass, 1)
    found = (upto <= (uniforms.double() * upto[:, -1])[:, None]).sum(1)
    prob = mass.gather(1, found[:, None])[:, 0] / upto[:, -1]
    return found.to(torch.int32), prob.float()


# ------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        names = ("uniforms", "temperature", "top_k", "top_p", "min_p")
        rows = [_exact_row(s["logits"][i].double().cpu().numpy(), *(s[k][i].item() for k in names)) for i in range(case["rows"])]
        return torch.tensor([r[0] for r in rows], dtype=torch.int32), torch.tensor([r[1] for r in rows], dtype=torch.float64)
    x, ids = s["x"].double(), s["ids"].cpu()
    y = torch.matmul(x, s["w"].double().T)
    for adapter in sorted(set(ids.tolist()) - {-1}):
        rows = torch.nonzero(ids == adapter)[:, 0].cuda()
        inner = torch.matmul(x[rows], s["a"][adapter].double().T)
        y[rows] += float(s["scale"][adapter]) * torch.matmul(inner, s["b"][adapter].double().T)
    return y


def _exact_row(logits, u, temperature, top_k, top_p, min_p):
    if temperature == 0:
        return int(np.argmax(logits)), 1.0
    weight = np.exp((logits - logits.max()) / temperature)
    order = np.lexsort((np.arange(len(logits)), -logits))
    count = len(order) if top_k <= 0 else min(top_k, len(order))
    if top_p < 1:
        reached = np.cumsum(weight[order])
        count = min(count, int(np.searchsorted(reached, top_p * reached[-1], side="left")) + 1)
    if min_p > 0:
        count = min(count, int(np.count_nonzero(logits - logits.max() >= temperature * np.log(min_p))))
    ids = np.sort(order[:count])
    sums = np.cumsum(weight[ids])
    at = int(np.searchsorted(sums, u * sums[-1], side="right"))
    return int(ids[at]), float(weight[ids[at]] / sums[-1])
