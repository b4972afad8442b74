"""Stored prefixes, forks and samples over 4-bit pages, where they meet other formats, full caches and many settings; two ranks; logits on the device."""
import json
import os
import subprocess
import sys
from dataclasses import replace
from pathlib import Path

import pytest
import torch

from _oracle import assert_tokens_equal_up_to_ties

from flyingfish_b200.engine.engine import DECODE_BUCKETS
from flyingfish_b200.engine.kv_cache import OutOfBlocks, PagedKVCache
from flyingfish_b200.engine.sampling import Sampling
from flyingfish_b200.loaders.safetensors_io import SafetensorsFile
from flyingfish_b200.ops import kv4_ops
from flyingfish_b200.utils.prefix_cache import restore_prefix, save_prefix
from test_kv4_engine import _load, _prompt


@pytest.mark.parametrize("order", [("bf16", "affine4"), ("affine4", "bf16")])
def test_one_store_holds_a_prompt_in_both_formats(tmp_path, order):
    """The formats share a directory of stored prefixes: each stores a prompt of its own there, and finds it again."""
    ids, want = _prompt(70), {}
    for kv_format in order + order:
        m = _load("cpu", kv_format=kv_format, prefix_cache=True, runtime_dir=str(tmp_path))
        first = m.prefill(ids)
        store, again = m.prefix_store(), kv_format in want
        assert (store.stored, store.hits) == ((0, 1) if again else (1, 0))
        got = [first] + [m.decode() for _ in range(3)]
        assert got == want.setdefault(kv_format, got)


@pytest.mark.parametrize("n", [64, 66, 127])
def test_stored_pages_hold_nothing_of_other_requests(tmp_path, n):
    """A block that was used before still holds another request's keys and values behind a prefix: they are not stored with it."""
    m = _load("cpu", capacity=256)
    kv = m.engine.kv
    for t in kv.k + kv.v:
        t.fill_(0x5A)
    seq = m.engine.add_sequence(_prompt(n))
    m.engine.prefill([seq])
    m.engine.decode([seq])
    kv.truncate(seq.seq_id, n)
    held = kv.seqs[seq.seq_id].blocks
    before = [t[held].clone() for t in kv.k + kv.v]
    pkg = save_prefix(m, seq, tmp_path / "pfx")
    assert all(torch.equal(t[held], w) for t, w in zip(kv.k + kv.v, before))
    f = SafetensorsFile(pkg / "kv.safetensors")
    try:
        for layer in range(kv.layers):
            for tag, cache, keys in (("k", kv.k[layer], True), ("v", kv.v[layer], False)):
                pages = f.tensor(f"layer.{layer}.{tag}")
                values = kv4_ops.page_values(pages, m.engine.model.d, keys).transpose(0, 1).flatten(1, 2)
                want = kv4_ops.page_values(cache[held], m.engine.model.d, keys).transpose(0, 1).flatten(1, 2)
                assert torch.equal(values[:, :n], want[:, :n]) and not values[:, n:].any()
                assert int((pages[-1] == 0x5A).sum()) <= pages[-1].numel() // 64       # (a code may be that by chance)
    finally:
        f.close()
    # and restored into a used block, tokens behind them stay
    m.reset()
    for t in kv.k + kv.v:
        t.fill_(0xA5)
    seq = restore_prefix(m, pkg)
    assert kv.seqs[seq.seq_id].length == n
    for cache, was, keys in zip(kv.k + kv.v, before, [True] * kv.layers + [False] * kv.layers):
        got, want = (kv4_ops.page_values(t, m.engine.model.d, keys).transpose(0, 1).flatten(1, 2)[:, :n] for t in (cache[kv.seqs[seq.seq_id].blocks], was))
        assert torch.equal(got, want)
        if n % 64:
            assert bool((cache[kv.seqs[seq.seq_id].blocks[-1]][:, kv4_ops.token_bytes(m.engine.model.d, keys)[n % 64:].flatten()] == 0xA5).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keys", [True, False])
def test_every_byte_of_a_page_is_a_tokens(dim, keys):
    at = kv4_ops.token_bytes(dim, keys)
    assert torch.equal(at.flatten().sort().values, torch.arange(kv4_ops.page_bytes(dim)))
    assert all(set(at[k, : dim // 2].tolist()) == set(kv4_ops._places(dim, keys)[0][k].tolist()) for k in range(64))


@pytest.mark.parametrize("kv_format", ["bf16", "affine4"])
def test_the_last_owner_of_a_shared_block_keeps_it_cpu(kv_format):
    """Sequences that were all taken back into a block that nobody else has: one of them needs no copy, and no free block for it."""
    kv = PagedKVCache(1, 1, 64, 4, kv_format=kv_format)
    kv.add_sequence(0)
    kv.reserve(0, 64)
    kv.commit(0, 64)
    kv.fork(0, 1)
    kv.fork(0, 2)
    for i in (0, 1, 2):
        kv.truncate(i, 30 + i)
    kv.add_sequence(3)
    kv.reserve(3, 64)
    assert kv.alloc.free_blocks == 2 and kv.blocks_wanted([(0, 1), (1, 1), (2, 1)]) == 2 == kv.blocks_wanted([(0, 1), (2, 20)]) and kv.blocks_wanted([(1, 60)]) == 2
    held, at, slots = kv.reserve_step([0, 1, 2])
    assert kv.alloc.shared == 0 == kv.alloc.free_blocks and len({int(s) // 64 for s in slots}) == 3 and [int(s) % 64 for s in slots] == [30, 31, 32]
    for i in range(4):
        kv.free_sequence(i)
    assert kv.alloc.free_blocks == 4


def test_a_step_over_forks_taken_back_needs_the_copies_that_are_made_cpu():
    m = _load("cpu")
    eng, ids = m.engine, _prompt(64)
    a = eng.add_sequence(ids)
    eng.prefill([a])
    b = eng.fork(a)
    for s in (a, b):
        eng.kv.truncate(s.seq_id, 30)
    eng.kv.add_sequence(99)
    eng.kv.reserve(99, 64 * (eng.kv.alloc.free_blocks - 1))
    assert eng.kv.alloc.free_blocks == 1
    eng._need_blocks([(a.seq_id, 1), (b.seq_id, 1)])
    eng.decode([a, b])
    assert eng.kv.alloc.free_blocks == 0 and a.output == b.output


def test_more_samples_than_a_decode_step_takes_cpu():
    """Samples are decoded in groups of what a step takes; the engine goes on afterwards."""
    m = _load("cpu")
    ids = _prompt(20)
    how = [Sampling(temperature=0.9, seed=s) for s in range(DECODE_BUCKETS[-1] + 3)]
    m.engine.kv = PagedKVCache(m.spec.layers, m.engine.kv.kv_heads, m.engine.kv.head_dim, 300, kv_format="affine4")
    got = m.generate_samples(ids, how, 3)
    assert [len(g) for g in got] == [3] * len(how) and not m.engine.poisoned
    for i in (0, 100, len(how) - 1):
        assert got[i] == m.engine.generate([ids], 3, sampling=how[i])[0]
    assert m.engine.kv.alloc.free_blocks == 300


def test_samples_that_the_cache_does_not_hold_leave_the_engine_usable_cpu():
    m = _load("cpu")
    ids, blocks = _prompt(65), m.engine.kv.num_blocks
    how = [Sampling(temperature=0.9, seed=s) for s in range(blocks + 2)]
    with pytest.raises(OutOfBlocks):
        m.generate_samples(ids, how, 3)
    assert not m.engine.poisoned and m.engine.kv.alloc.free_blocks == blocks and not m.engine.seqs
    assert len(m.generate_samples(ids, how[:3], 3)) == 3


def test_two_ranks_over_4_bit_pages_cpu(tmp_path):
    """Each rank's pages hold its share of the heads (one at least); tokens are those of one rank, up to ties (the ranks' sums are added in another order)."""
    prompts, out = [_prompt(100), _prompt(9, 12)], tmp_path / "out.json"
    (tmp_path / "in.json").write_text(json.dumps(prompts))
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port", "29541",
           str(Path(__file__).resolve().parent / "kv4_tp_worker.py"), str(tmp_path / "in.json"), str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600, env=dict(os.environ, OMP_NUM_THREADS="2"))
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    got, m = json.loads(out.read_text()), _load("cpu", capacity=256)
    assert got["page"][1:] == [max(1, m.engine.kv.kv_heads // 2), kv4_ops.page_bytes(m.engine.model.d)]
    for p, want, tokens in zip(prompts, m.generate_batch(prompts, 8), got["tokens"]):
        assert_tokens_equal_up_to_ties(m, p, want, tokens)


def _plain(seq):
    """The sequence without its settings, which a forward over given tokens refuses."""
    return replace(seq, draws=None)


# ------------------------------------------------------------------------------------------
# on the device
# ------------------------------------------------------------------------------------------
# Two computations of the same model quantise keys and values whose last bits differ: a code next to a border falls on either side of it. Were all codes so, an element
# would be off by two independent errors of half a step (1 / 15 of a group's span, some four standard deviations, over sqrt(12): 0.08 of a standard deviation each), 0.11 in
# the root mean square, and what is made of them as much at most where attention's average takes nothing off it. Attention over the wrong pages moves these logits by 1 and more.
APART = 0.11


def _off(x, y):
    return float((x.float().cpu() - y.float().cpu()).norm() / y.float().norm().cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 64, 300])
def test_logits_are_those_of_the_host(n):
    """Of a prompt in portions, of rows behind it and of a decode step in a captured graph, and the pages of the last layer, whose keys depend on every attention before."""
    got, want, kept = [], [], []
    for device, out in (("cuda", got), ("cpu", want)):
        m = _load(device, graph=device == "cuda", capacity=512)
        eng = m.engine
        other, seq = eng.add_sequence(_prompt(90, 5)), eng.add_sequence(_prompt(n))
        eng.prefill([other, seq], chunk=70)
        out.append(eng.forward_rows(seq, _prompt(40, 3)).clone())                    # prompt rows, in tiles on the device
        out.append(eng.forward_rows(seq, _prompt(3, 4)).clone())                     # a few
        for token in _prompt(66, 6):                                                 # given tokens, so that both sides see the same ones
            other.pending, seq.pending = 7, token
            _, logits, _ = eng._launch_decode([other, seq])
            logits = logits[1:2].cpu()                                               # (the next step writes this one's host buffer)
            for s in (other, seq):
                eng.kv.commit(s.seq_id, 1)
        out.append(logits)
        kv, layer = eng.kv, m.spec.layers - 1
        slots = torch.tensor([kv.seqs[seq.seq_id].blocks[p // 64] * 64 + p % 64 for p in range(n + 66)], dtype=torch.int32, device=device)
        out += list(kv4_ops.read_kv4(kv.k[layer], kv.v[layer], slots, eng.model.d))
        kept.append(m)
    assert kept[0].engine.stats["graph_replays"] == 66
    for x, y in zip(got, want):
        assert x.shape == y.shape and bool(torch.isfinite(x).all()) and _off(x, y) < APART
    assert _off(got[0][1:], want[0][:-1]) > 3 * APART                                # rows of neighbouring places differ by far more


@pytest.mark.gpu
@pytest.mark.parametrize("kv_format", ["bf16", "affine4"])
def test_each_sample_starts_from_a_separate_requests_logits(kv_format):
    m = _load("cuda", kv_format=kv_format, graph=True, capacity=512)
    eng, ids = m.engine, _prompt(200)
    alone = eng.add_sequence(ids)
    eng.prefill([alone])
    eng.kv.truncate(alone.seq_id, len(ids) - 1)
    want = eng.forward_rows(alone, ids[-1:]).clone()
    whole = eng.add_sequence(ids)
    eng.prefill([whole])
    forks = [eng.fork(whole, Sampling(temperature=0.9, seed=s), again=True) for s in (3, 4, 5)]
    for f in forks:
        assert _off(eng.forward_rows(_plain(f), ids[-1:]), want) < APART
    assert len(eng.prefill(forks)) == 3
