"""Requests with settings and adapters of their own, through the engine, the scheduler, the server and the command line: low-rank adapters
beside the model's projections, tokens drawn per request, both in one batch."""
import asyncio
import json

import numpy as np
import pytest
import torch
from aiohttp.test_utils import TestClient, TestServer

from flyingfish_b200 import cli
from flyingfish_b200.api import Model, generate_plain
from flyingfish_b200.config import Settings
from flyingfish_b200.engine.engine import Span
from flyingfish_b200.engine.sampling import BLOCK, Draws, Sampling, philox_uniforms
from flyingfish_b200.engine.scheduler import Request, Scheduler
from flyingfish_b200.loaders.adapters import AdapterError, build_adapters, read_adapter
from flyingfish_b200.loaders.safetensors_io import save_safetensors
from flyingfish_b200.loaders.tokenizer import ByteTokenizer
from flyingfish_b200.models.weights import TPInfo
from flyingfish_b200.ops import ref, sample_ops
from flyingfish_b200.serve.backend import Backend, MtpBackend
from flyingfish_b200.serve.http import Server

ALL = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")
TINY = {"q_proj": (512, 512), "k_proj": (128, 512), "v_proj": (128, 512), "o_proj": (512, 512), "gate_proj": (1024, 512), "up_proj": (1024, 512),
        "down_proj": (512, 1024)}


def _entries(rank, seed, projs=ALL, scale=2.0, layers=(0, 1), dtype=torch.bfloat16):
    """Matrices whose products are about as large as the tiny model's weights (N(0, 0.02))."""
    g = torch.Generator().manual_seed(seed)
    return {(l, p): ((torch.randn(rank, TINY[p][1], generator=g) * 0.1).to(dtype), (torch.randn(TINY[p][0], rank, generator=g) * 0.1 * rank ** -0.5).to(dtype),
                     scale) for l in layers for p in projs}


ADAPTERS = {"poet": lambda: _entries(8, 1), "clerk": lambda: _entries(40, 2, ("q_proj", "v_proj"), 1.0), "cook": lambda: _entries(3, 3, ("gate_proj", "o_proj"), 0.5, (1,))}


def _load(device="cpu", adapters=ADAPTERS, **kw):
    kw = {"capacity": 256, "max_batch": 4, **kw}
    return Model.load("tiny-llama", Settings(**kw), device=device, seed=0, adapters={n: e() for n, e in adapters.items()} or None)


def _prompt(n, seed):
    return torch.randint(1, 2000, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _write_adapter(path, entries, config=None, names="base_model.model.model.layers.{l}.{m}.{p}.lora_{s}.weight"):
    path.mkdir()
    tensors = {}
    for (l, p), (a, b, _) in entries.items():
        m = "mlp" if p in ("gate_proj", "up_proj", "down_proj") else "self_attn"
        for s, t in (("A", a), ("B", b)):
            tensors[names.format(l=l, m=m, p=p, s=s)] = t
    save_safetensors(path / "adapter_model.safetensors", tensors)
    (path / "adapter_config.json").write_text(json.dumps({"peft_type": "LORA", "r": 8, "lora_alpha": 16, **(config or {})}))
    return path


# ------------------------------------------------------------------------------------------
# settings and random numbers
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seed", [0, 1, 0x9E3779B97F4A7C15, (1 << 64) - 1])
def test_numbers_are_those_of_the_counter_based_generator(seed):
    for start, n in ((0, 9), (3, 5), (1021, 4), ((1 << 34) + 1, 6)):
        got = philox_uniforms(seed, start, n)
        want = []
        for i in range(start, start + n):
            c = i // 4
            word = ref.philox4x32_10((seed & 0xFFFFFFFF, seed >> 32), (c & 0xFFFFFFFF, c >> 32, 0, 0))[i % 4]
            want.append((word >> 8) / 16777216.0)
        assert got.dtype == np.float32 and got.tolist() == want
    d = Draws(Sampling(seed=seed))
    asked = [5, BLOCK - 1, BLOCK, 3 * BLOCK + 7, 5]
    assert [float(d.uniform(i)) for i in asked] == [float(philox_uniforms(seed, i, 1)[0]) for i in asked]


@pytest.mark.parametrize("bad", [{"temperature": -1}, {"temperature": float("nan")}, {"temperature": "1"}, {"temperature": True}, {"temperature": 10 ** 400}, {"top_k": -1},
                                 {"top_k": 1.5}, {"top_k": 1 << 31}, {"top_p": 0}, {"top_p": 1.01}, {"min_p": -0.1}, {"min_p": 2}, {"seed": -1},
                                 {"seed": 1 << 64}, {"seed": None}])
def test_settings_are_checked(bad):
    with pytest.raises(ValueError):
        Sampling(**bad)


def test_a_plain_step_uploads_what_it_did():
    eng = _load().engine
    fb = eng._decode_batch(4)
    seqs = [eng.add_sequence([1, 2, 3 + i]) for i in range(3)]
    eng.prefill(seqs)
    eng.decode(seqs)
    assert fb.host.numel() == fb.dev.numel() == fb.layout.total          # whoever stages plain steps by hand copies these whole
    assert fb.h2d_bytes() == 4 * fb.layout.total < 4 * fb.layout.full and fb.adapters is None and not fb.sampled
    s = eng.add_sequence([1, 2, 9], adapter="poet", sampling=Sampling(0.5))
    eng.prefill([s])
    eng.decode([seqs[0], s])
    fb = eng._decode_batch(2)
    assert fb.h2d_bytes() == 4 * fb.layout.full and fb.adapter_ids.tolist() == [-1, 0] and fb.temperature.tolist() == [0.0, 0.5]
    eng.free_sequence(s.seq_id)
    eng.decode(seqs[:2])
    assert fb.adapters is None and not fb.sampled


# ------------------------------------------------------------------------------------------
# adapter directories
# ------------------------------------------------------------------------------------------
def test_an_adapter_directory_is_read(tmp_path):
    e = _entries(8, 5)
    got = read_adapter(_write_adapter(tmp_path / "a", e))
    assert set(got) == set(e) and all(torch.equal(got[k][i], e[k][i]) for k in e for i in (0, 1)) and all(v[2] == 2.0 for v in got.values())
    got = read_adapter(_write_adapter(tmp_path / "b", e, {"use_rslora": True, "alpha_pattern": {"q_proj": 4, "layers.1.mlp.up_proj": 24}},
                                      "model.layers.{l}.{m}.{p}.lora_{s}.default.weight"))
    assert got[0, "q_proj"][2] == 4 / 8 ** 0.5 and got[1, "up_proj"][2] == 24 / 8 ** 0.5 and got[0, "up_proj"][2] == 16 / 8 ** 0.5


@pytest.mark.parametrize("config", [{"peft_type": "IA3"}, {"bias": "all"}, {"modules_to_save": ["lm_head"]}, {"use_dora": True}, {"fan_in_fan_out": True},
                                    {"lora_alpha": "x"}, {"lora_alpha": float("inf")}, {"alpha_pattern": {".*q_proj": 4}}, {"layer_replication": [[0, 2]]}])
def test_adapter_kinds_without_a_place_are_refused(tmp_path, config):
    with pytest.raises(AdapterError):
        read_adapter(_write_adapter(tmp_path / "a", _entries(4, 1), config))


@pytest.mark.parametrize("init", ["pissa", "pissa_niter_16", "olora", "CorDA", "loftq"])
def test_adapters_of_a_changed_base_are_refused(tmp_path, init):
    with pytest.raises(AdapterError, match="convert"):
        read_adapter(_write_adapter(tmp_path / "a", _entries(4, 1), {"init_lora_weights": init}))
    assert read_adapter(_write_adapter(tmp_path / "b", _entries(4, 1), {"init_lora_weights": True}))
    assert read_adapter(_write_adapter(tmp_path / "c", _entries(4, 1), {"init_lora_weights": "gaussian"}))


def test_broken_adapters_are_refused(tmp_path):
    with pytest.raises(AdapterError):
        read_adapter(tmp_path)
    e = _entries(4, 1)
    with pytest.raises(AdapterError, match="embed"):
        read_adapter(_write_adapter(tmp_path / "a", e, names="model.embed_tokens{l}{p}.lora_{s}.weight"))
    lone = tmp_path / "b"
    lone.mkdir()
    (lone / "adapter_config.json").write_text("{}")
    save_safetensors(lone / "adapter_model.safetensors", {"layers.0.mlp.up_proj.lora_A.weight": e[0, "up_proj"][0]})
    with pytest.raises(AdapterError, match="up_proj"):
        read_adapter(lone)
    a, b, s = e[0, "q_proj"]
    bad = a.clone()
    bad[0, 0] = float("nan")
    net = _load(adapters={}).engine.model
    for entry, at in (((a, b[:-1], s), (0, "q_proj")), ((a[:, 1:], b, s), (0, "q_proj")), ((a, b, s), (2, "q_proj")), ((bad, b, s), (0, "q_proj")),
                      ((torch.zeros(400, 512), torch.zeros(512, 400), s), (0, "q_proj"))):
        with pytest.raises(AdapterError):
            build_adapters(net, {"x": {at: entry}})


@pytest.mark.parametrize("prefix", ["base_model.model.vision_tower.encoder", "model.visual.transformer", "encoder", "model.language_model.visual"])
def test_matrices_of_another_tower_are_refused(tmp_path, prefix):
    with pytest.raises(AdapterError, match="none of the decoder"):
        read_adapter(_write_adapter(tmp_path / "a", _entries(4, 1), names=prefix + ".layers.{l}.{m}.{p}.lora_{s}.weight"))


@pytest.mark.parametrize("prefix", ["base_model.model.model", "base_model.model.model.language_model", "language_model.model", "model"])
def test_a_decoders_names_are_known_with_what_stands_before_them(tmp_path, prefix):
    got = read_adapter(_write_adapter(tmp_path / "a", _entries(4, 1), names=prefix + ".layers.{l}.{m}.{p}.lora_{s}.weight"))
    assert set(got) == set(_entries(4, 1))


@pytest.mark.parametrize("data", [b"", b"1234567", b"\xff" * 64, (8).to_bytes(8, "little") + b"nonsense"])
def test_files_that_hold_no_matrices_are_refused(tmp_path, data):
    (tmp_path / "adapter_config.json").write_text("{}")
    (tmp_path / "adapter_model.safetensors").write_bytes(data)
    with pytest.raises(AdapterError, match="adapter_model"):
        read_adapter(tmp_path)
    with pytest.raises(SystemExit):
        cli.main(["--model", "tiny-llama", "--cpu", "generate", "--tokens", "1", "--max-new-tokens", "1", "--adapter", str(tmp_path)])


def test_a_matrix_named_twice_is_refused(tmp_path):
    path = tmp_path / "a"
    path.mkdir()
    (path / "adapter_config.json").write_text("{}")
    a, b, _ = _entries(4, 1)[0, "q_proj"]
    save_safetensors(path / "adapter_model.safetensors", {f"{p}layers.0.self_attn.q_proj.lora_{s}.weight": t for p in ("model.", "base_model.model.model.") for s, t in (("A", a), ("B", b))})
    with pytest.raises(AdapterError, match="second"):
        read_adapter(path)


@pytest.mark.parametrize("shape", ["tiny-hybrid", "deepseek-v3-tiny"])
def test_models_without_the_plain_projections_are_refused(shape):
    with pytest.raises(AdapterError):
        Model.load(shape, Settings(capacity=128, max_batch=2), device="cpu", adapters={"x": {(0, "q_proj"): (torch.zeros(4, 8), torch.zeros(8, 4), 1.0)}})


def test_a_mixture_takes_adapters_in_its_attention():
    spec = Model.load("tiny-moe", Settings(capacity=64, max_batch=2), device="cpu").spec
    a = lambda n: (torch.randn(4, 256, generator=torch.Generator().manual_seed(n)) * 0.2, torch.randn(n, 4, generator=torch.Generator().manual_seed(n)) * 0.2, 1.0)
    m = Model.load("tiny-moe", Settings(capacity=64, max_batch=2), device="cpu", adapters={"x": {(0, "q_proj"): a(256), (0, "k_proj"): a(128)}})
    e = m.engine.generate([[1, 2, 3], [1, 2, 3]], 8, adapter=["x", None])
    assert e[1] == m.engine.generate([[1, 2, 3]], 8)[0] and e[0] != e[1] and spec.moe is not None
    with pytest.raises(AdapterError, match="up_proj"):
        Model.load("tiny-moe", Settings(capacity=64, max_batch=2), device="cpu", adapters={"x": {(0, "up_proj"): (torch.zeros(4, 256), torch.zeros(512, 4), 1.0)}})


# ------------------------------------------------------------------------------------------
# adapters in the model
# ------------------------------------------------------------------------------------------
def _logits(model, ids, adapter=None):
    eng = model.engine
    s = eng.add_sequence(ids, adapter=adapter)
    fb = eng._fill_spans([Span(s, ids, [len(ids) - 1])])
    out = eng.model.forward(fb, eng.kv, return_logits=True).float().cpu()[0]
    eng.free_sequence(s.seq_id)
    return out


@pytest.mark.parametrize("name", list(ADAPTERS))
def test_adapters_are_merged_weights(name):
    """In FP32, logits with an adapter are those of the weights with scale B A added. Two chains of a dozen products of at most 1024 terms each lose
    1024 * 2^-24 = 2^-14 of a product's size at worst, together less than 2^-10 of the logits' scale; the adapters change them by far more."""
    m = _load(dtype="fp32")
    ids = _prompt(23, 7)
    got, base = _logits(m, ids, name), _logits(m, ids)
    plain = _load(adapters={}, dtype="fp32")
    assert torch.equal(base, _logits(plain, ids))
    for (l, p), (a, b, s) in ADAPTERS[name]().items():
        lw, d = plain.engine.model.w.layers[l], s * b.float() @ a.float()
        if p in ("q_proj", "k_proj", "v_proj"):
            at = {"q_proj": 0, "k_proj": 512, "v_proj": 640}[p]
            lw.wqkv[at: at + d.shape[0]] += d
        elif p in ("gate_proj", "up_proj"):
            lw.wgu.view(-1, 2, 64, 512)[:, int(p == "up_proj")] += d.view(-1, 64, 512)
        else:
            getattr(lw, {"o_proj": "wo", "down_proj": "wdown"}[p]).add_(d)
    want = _logits(plain, ids)
    scale = want.abs().max()
    assert (got - want).abs().max() <= 2.0 ** -10 * scale < (want - base).abs().max()


def test_parts_of_no_whole_64_columns_share_one_part():
    """A fused projection of 3 x 32 columns goes through one part's stack."""
    from flyingfish_b200.loaders.adapters import _one_part
    from flyingfish_b200.ops import lora_ops
    g = torch.Generator().manual_seed(0)
    new = lambda *s: torch.randn(*s, generator=g)
    parts = [(new(3, 32), new(32, 3), 0.5), None, (new(2, 32), new(16, 2), 2.0)]
    st = lora_ops.pack_stack(_one_part([parts, [None] * 3], [32, 16, 16]), 32, [64], "cpu", torch.float32)
    x, w = new(4, 32), new(64, 32)
    y = lora_ops.linear_lora(x, w, st, torch.tensor([0, -1, 1, 0], dtype=torch.int32))
    d = torch.cat([0.5 * parts[0][1] @ parts[0][0], torch.zeros(16, 32), 2.0 * parts[2][1] @ parts[2][0]])
    want = torch.stack([x[0] @ (w + d).T, x[1] @ w.T, x[2] @ w.T, x[3] @ (w + d).T])
    assert torch.allclose(y, want, rtol=1e-5, atol=1e-4)              # 64 terms: 64 * 2^-24 = 4e-6 of sums of up to 20


# ------------------------------------------------------------------------------------------
# a batch of both
# ------------------------------------------------------------------------------------------
HOW = [(None, None), (Sampling(1.0, seed=11), "poet"), (Sampling(0.8, top_k=20, seed=12), None), (None, "clerk"),
       (Sampling(2.0, top_p=0.9, min_p=0.02, seed=(1 << 63) + 5), "cook"), (Sampling(1.5, seed=11), "poet"), (Sampling(0), None)]


def _mixed(model, tokens=12, chunk=16, midway=None):
    sched = Scheduler(model.engine, token_budget=chunk)
    reqs = [sched.submit(Request(prompt=_prompt(5 + 9 * i, 50 + i), max_tokens=tokens, sampling=h, adapter=a)) for i, (h, a) in enumerate(HOW)]
    it = 0
    while sched.has_work():
        sched.step()
        it += 1
        if midway is not None and it in midway and sched.running:
            sched._preempt_youngest()
    assert all(r.state == "finished" and len(r.output) == tokens for r in reqs)
    return [r.output for r in reqs]


def test_a_request_gives_the_same_tokens_alone_and_among_others():
    m = _load(dtype="fp32")
    got = _mixed(m)
    for i, (h, a) in enumerate(HOW):
        alone = m.engine.generate([_prompt(5 + 9 * i, 50 + i)], 12, sampling=h, adapter=a)[0]
        assert alone == got[i], f"request {i}"
    assert _load(dtype="fp32", adapters={}).engine.generate([_prompt(5, 50)], 12)[0] == got[0]
    # settings matter: without them the tokens are others
    assert got[6] == m.engine.generate([_prompt(59, 56)], 12)[0] and got[2] != m.engine.generate([_prompt(23, 52)], 12)[0]


def test_a_preempted_request_goes_on_with_its_numbers():
    m = _load(dtype="fp32")
    assert _mixed(m, midway=(6, 9, 13)) == _mixed(m)


def test_drawn_tokens_are_those_of_the_operator():
    """Every token is the operator's answer to the step's logits, the request's settings and the number of its place in the sequence."""
    m = _load(dtype="fp32")
    eng, how = m.engine, Sampling(1.3, top_k=50, top_p=0.95, seed=77)
    ids = _prompt(9, 3)
    s = eng.add_sequence(ids, sampling=how, adapter="poet")
    want = []
    for i in range(6):
        if i == 0:
            eng.prefill([s])
        else:
            eng.decode([s])
        lg = eng.model.last_logits
        row = lambda v, t: torch.tensor([v], dtype=t)
        tok, _ = sample_ops.sample_tokens(lg[:1], row(float(philox_uniforms(77, 9 + i, 1)[0]), torch.float32), row(1.3, torch.float32), row(50, torch.int32),
                                          row(0.95, torch.float32), row(0.0, torch.float32))
        want.append(int(tok[0]))
    assert s.output == want and len(set(want)) > 2


def test_fed_tokens_take_the_adapter_and_nothing_is_drawn():
    m = _load(dtype="fp32")
    ids = _prompt(12, 8)
    if not m.engine.mixed_batches:
        m.engine.mixed_batches = True                # single tokens replay the decode step, which every model has
    s = m.engine.add_sequence(ids[:1], adapter="poet", sampling=Sampling(5.0, seed=1))
    for t in ids:
        lg = m.engine.feed([Span(s, [t], [0])])
    want = _logits(m, ids, "poet")
    assert (lg[0] - want).abs().max() <= 2.0 ** -10 * want.abs().max()            # the bound of the merged weights


def test_what_compares_with_greedy_tokens_refuses_such_sequences():
    eng = _load().engine
    with pytest.raises(ValueError, match="no adapter"):
        eng.add_sequence([1], adapter="nobody")
    with pytest.raises(ValueError, match="no adapter"):
        Scheduler(eng).submit(Request(prompt=[1], max_tokens=1, adapter="nobody"))
    with pytest.raises(ValueError, match="one per prompt"):
        eng.generate([[1], [2]], 2, sampling=[None])
    for kw in ({"sampling": Sampling()}, {"adapter": "poet"}):
        s = eng.add_sequence([1, 2, 3], **kw)
        eng.prefill([s])
        with pytest.raises(ValueError, match="not available"):
            eng.verify([s], [[1, 2]])
        with pytest.raises(ValueError, match="not available"):
            eng.verify_tree(s, [s.pending], [0], [1])
        with pytest.raises(ValueError, match="not available"):
            eng.forward_rows(s, [1])
        assert not eng.poisoned and len(eng.decode([s])) == 1
        eng.free_sequence(s.seq_id)
    tp = eng.model.w.tp
    try:
        eng.model.w.tp = TPInfo(0, 2)
        with pytest.raises(ValueError, match="tensor"):
            eng.add_sequence([1], sampling=Sampling())
        with pytest.raises(ValueError, match="tensor"):
            Scheduler(eng).submit(Request(prompt=[1], max_tokens=1, sampling=Sampling()))
        with pytest.raises(AdapterError, match="tensor"):
            build_adapters(eng.model, {"x": _entries(4, 1)})
    finally:
        eng.model.w.tp = tp
    with pytest.raises(AdapterError, match="the model's name"):
        Model.load("tiny-llama", Settings(capacity=64), device="cpu", adapters={"tiny-llama": _entries(4, 1)})


# ------------------------------------------------------------------------------------------
# server and command line
# ------------------------------------------------------------------------------------------
def test_greedy_settings_ask_for_nothing():
    """Temperature 0 is the plain path, with tensor parallelism too."""
    eng = _load().engine
    tp = eng.model.w.tp
    try:
        eng.model.w.tp = TPInfo(0, 2)
        s = eng.add_sequence([1, 2], sampling=Sampling(0))
        assert s.draws is None and not s.special
        assert Scheduler(eng).submit(Request(prompt=[1], max_tokens=1, sampling=Sampling(0.0))).sampling.temperature == 0
    finally:
        eng.model.w.tp = tp


class Numbers(ByteTokenizer):
    """Ids as text, so that answers show the tokens."""

    def decode(self, ids, skip_special_tokens=True):
        return "".join(f"{i} " for i in ids)


def _serve(model, go, sampling=True, adapters=tuple(ADAPTERS)):
    async def main():
        backend = Backend(model.engine, eos_ids=(257,))
        backend.start()
        srv = Server(backend, Numbers(model.spec.vocab), "tiny-llama", None, capacity=256, allow_sampling=sampling, adapters=adapters)
        client = TestClient(TestServer(srv.app()))
        await client.start_server()
        try:
            return await go(client)
        finally:
            await client.close()
            backend.shutdown()
            model.engine.reset()
    return asyncio.run(main())


async def _post(client, status=200, **body):
    r = await client.post("/v1/completions", json={"prompt": [5, 6, 7, 8], "max_tokens": 10, **body})
    b = await r.json()
    assert r.status == status, b
    return b if status != 200 else b["choices"][0]["text"]


def test_the_server_draws_by_the_request():
    m = _load(dtype="fp32")

    async def go(client):
        greedy = await _post(client)
        assert await _post(client, temperature=0, top_p=0.5, top_k=3) == greedy
        hot = dict(temperature=3.0, seed=42)
        a, b, c, d = await asyncio.gather(_post(client, **hot), _post(client, temperature=3.0, seed=43), _post(client, model="poet", **hot), _post(client, **hot))
        assert a == d and len({a, b, c, greedy}) == 4
        assert await _post(client, top_k=1, **hot) == greedy == await _post(client, min_p=1, **hot)
        assert await _post(client, top_k=-1, min_p=0, **hot) == a
        assert await _post(client, temperature=3.0) != await _post(client, temperature=3.0)            # a seed of its own for each
        for bad in ({"temperature": -1}, {"temperature": "hot"}, {"temperature": 1, "top_p": 0}, {"temperature": 1, "top_k": 2.5}, {"min_p": 3}, {"seed": -5},
                    {"seed": 1.5}, {"n": 2}, {"logit_bias": {"1": 2}}, {"presence_penalty": 1}, {"stop": "x"}, {"best_of": 2}):
            await _post(client, 400, **bad)
        await _post(client, 404, model="nobody")
        r = await client.post("/v1/completions", json={"prompt": [5], "max_tokens": 1, "model": "poet"})
        assert (await r.json())["model"] == "poet"
        return greedy, await _post(client, model="poet")
    base, poet = _serve(m, go)
    assert base != poet

    async def strict(client):
        assert await _post(client) == base and await _post(client, model="poet") == poet
        for bad in ({"temperature": 1}, {"seed": 4}, {"min_p": 0.5}):
            await _post(client, 400, **bad)
    _serve(m, strict, sampling=False)


def test_speculation_serves_greedy_requests_only():
    m = Model.load("deepseek-v3-tiny", Settings(capacity=128, max_batch=2), device="cpu")
    backend = MtpBackend(m, 1)
    for kw in ({"allow_sampling": True}, {"adapters": ("x",)}):
        with pytest.raises(ValueError, match="greedy"):
            Server(backend, ByteTokenizer(m.spec.vocab), "x", None, **kw)


def test_speculation_takes_no_other_request():
    backend = MtpBackend(Model.load("deepseek-v3-tiny", Settings(capacity=128, max_batch=2), device="cpu"), 1)

    async def add(**kw):
        return backend.add_request([1, 2, 3], 4, **kw)
    for kw in ({"sampling": Sampling(0.5)}, {"adapter": "x"}):
        with pytest.raises(ValueError, match="greedy"):
            asyncio.run(add(**kw))
    assert not backend._inflight
    req, _ = asyncio.run(add(sampling=Sampling(0.0)))
    assert req.prompt == [1, 2, 3]


def test_the_command_line_draws_and_adapts(tmp_path, capsys):
    where = str(_write_adapter(tmp_path / "poet", _entries(8, 1)))

    def run(*extra):
        assert cli.main(["--model", "tiny-llama", "--cpu", "--capacity", "64", "generate", "--tokens", "5,6,7", "--max-new-tokens", "8", "--ignore-eos", *extra]) == 0
        return json.loads(capsys.readouterr().out)
    plain, drawn = run(), run("--temperature", "3", "--sample-seed", "4")
    assert drawn["generated_ids"] == run("--temperature", "3", "--sample-seed", "4")["generated_ids"] != plain["generated_ids"]
    assert drawn["sampling"] == {"temperature": 3.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "seed": 4} and "sampling" not in plain
    got = run("--adapter", where)
    m = Model.load("tiny-llama", Settings(capacity=64), device="cpu", adapters={"a": where})
    assert got["adapter"] == where and got["generated_ids"] == generate_plain(m, [5, 6, 7], 8, ignore_eos=True, adapter="a").ids != plain["generated_ids"]


@pytest.mark.parametrize("flags", [["--top-k", "5"], ["--temperature", "-1"], ["--temperature", "1", "--top-p", "0"], ["--temperature", "1", "--mtp", "2"],
                                   ["--adapter", "/nowhere"]])
def test_the_command_line_refuses(flags):
    with pytest.raises(SystemExit):
        cli.main(["--model", "tiny-llama", "--cpu", "generate", "--tokens", "1", "--max-new-tokens", "2", *flags])


@pytest.mark.parametrize("flags", [["--adapter", "x"], ["--adapter", "=d"], ["--adapter", "a=b", "--adapter", "a=c"], ["--allow-sampling", "--mtp", "1"],
                                   ["--adapter", "a=b", "--mtp", "1"], ["--adapter", "a=/nowhere"]])
def test_the_server_flags_are_checked(flags):
    with pytest.raises(SystemExit):
        cli.main(["--model", "tiny-llama", "--cpu", "serve", *flags])


# ------------------------------------------------------------------------------------------
# GPU
# ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 23, 150])
def test_adapted_logits_match_the_cpu_oracle(rows):
    """The tolerance is that of the plain model's comparison: BF16 activations on both sides, rounded at different places."""
    cpu, gpu = _load(), _load("cuda:0")
    ids = _prompt(rows, 9)
    for name in [None, *ADAPTERS]:
        want, got = _logits(cpu, ids, name), _logits(gpu, ids, name)
        assert (want - got).abs().max() < 0.05 * max(want.abs().max(), 1.0), name


def _fed(device, names, **kw):
    """Logits of decode rows of several adapters."""
    m = _load(device, **kw)
    m.engine.mixed_batches = True
    seqs = [m.engine.add_sequence(_prompt(3, 60 + i)[:1], adapter=n) for i, n in enumerate(names)]
    for step in range(3):
        out = m.engine.feed([Span(s, [_prompt(3, 60 + i)[step]], [0]) for i, s in enumerate(seqs)])
    return out.float().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_adapted_decode_matches_the_cpu_oracle(graph):
    names = ["poet", None, "cook", "clerk"]
    want, got = _fed("cpu", names), _fed("cuda:0", names, graph=graph)
    assert (want - got).abs().max() < 0.05 * max(want.abs().max(), 1.0)


@pytest.mark.gpu
def test_replayed_steps_give_the_eager_tokens():
    got = [_mixed(_load("cuda:0", graph=g, max_batch=8), tokens=16) for g in (False, True)]
    assert got[0] == got[1]
    m = _load("cuda:0", graph=True, max_batch=8)
    assert _mixed(m, tokens=16) == got[0] == _mixed(m, tokens=16)
    kinds = {k[2:] for k in m.engine.graphs if k[1] == 1}
    assert (True, True) in kinds


@pytest.mark.gpu
def test_drawn_tokens_of_a_captured_step_are_the_oracles():
    """The ids of a replayed step are those of its logits in 64 bits, row by row, and greedy rows beside them the largest."""
    m = _load("cuda:0", graph=True)
    eng = m.engine
    how = [Sampling(1.0, seed=5), None, Sampling(0.7, top_k=9, top_p=0.8, seed=6), Sampling(4.0, min_p=0.2, seed=7)]
    seqs = [eng.add_sequence(_prompt(6 + i, 20 + i), sampling=h, adapter=a) for i, (h, a) in enumerate(zip(how, ("poet", None, "cook", None)))]
    eng.prefill(seqs)
    for step in range(8):
        at = [eng.kv.seqs[s.seq_id].length + 1 for s in seqs]
        got = eng.decode(seqs)
        g = eng.graphs[4, 1, True, True]
        for i, h in enumerate(how):
            lg = g.logits[i: i + 1].cpu()
            if h is None:
                assert got[i] == int(lg[0].float().argmax())
                continue
            row = lambda v, t=torch.float32: torch.tensor([v], dtype=t)
            want, _ = ref.sample_tokens(lg, row(float(philox_uniforms(h.seed, at[i], 1)[0])), row(h.temperature), row(h.top_k, torch.int32), row(h.top_p),
                                        row(h.min_p))
            assert got[i] == int(want[0]), (step, i)


@pytest.mark.gpu
def test_plain_sequences_keep_their_tokens_after_a_mixed_batch():
    """Greedy sequences of the base model, before, and beside and after others: with nothing special alive the old graphs run."""
    m = _load("cuda:0", graph=True)
    ids = [_prompt(8, 30), _prompt(17, 31)]
    first = m.engine.generate(ids, 12)
    m.engine.generate([*ids, _prompt(5, 32)], 12, sampling=[None, None, Sampling(seed=3)], adapter=[None, None, "poet"])
    assert m.engine.generate(ids, 12) == first == _load("cuda:0", adapters={}, graph=True).engine.generate(ids, 12)
