"""Low-rank adapters (LoRA) of a decoder: the published adapter directories (``adapter_config.json`` + ``adapter_model.safetensors``) and the stacks
that a model's layers read (``ops/lora_ops.py``).

An adapter names the projections it changes (``...layers.N.self_attn.q_proj.lora_A.weight`` ...); q, k and v, and gate and up, are one product
each in this framework, so their adapters become the parts of one stack."""
from __future__ import annotations

import json
import math
import re
from dataclasses import dataclass, field
from pathlib import Path

import torch

from ..config import ModelSpec
from ..ops import lora_ops
from .safetensors_io import SafetensorsFile

PROJECTIONS = {"self_attn": ("q_proj", "k_proj", "v_proj", "o_proj"), "mlp": ("gate_proj", "up_proj", "down_proj")}
REBASED = ("pissa", "olora", "corda", "loftq")          # initialisations that leave the model without what the adapter begins with
FILES = ("adapter_config.json", "adapter_model.safetensors")
# a decoder's own layers: not those of a tower that a larger model has beside it, whose names end alike
_NAME = re.compile(r"^(?:base_model\.)?(?:model\.|language_model\.)*layers\.(\d+)\.(self_attn|mlp)\.(\w+)\.lora_([AB])(?:\.default)?\.weight$")

Entries = dict[tuple[int, str], tuple[torch.Tensor, torch.Tensor, float]]      # (layer, projection) -> A [r, K], B [N, r], scale


class AdapterError(ValueError):
    pass


@dataclass
class LayerStacks:
    """One layer's stacks; None where no adapter changes the projection."""
    qkv: lora_ops.AdapterStack | None = None
    o: lora_ops.AdapterStack | None = None
    gu: lora_ops.AdapterStack | None = None
    down: lora_ops.AdapterStack | None = None


@dataclass
class AdapterSet:
    """The adapters a model is loaded with. ``index`` gives the id that a batch's rows carry."""
    names: list[str]
    layers: list[LayerStacks]
    index: dict[str, int] = field(init=False)

    def __post_init__(self) -> None:
        self.index = {n: i for i, n in enumerate(self.names)}

    def nbytes(self) -> int:
        return sum(s.nbytes() for l in self.layers for s in (l.qkv, l.o, l.gu, l.down) if s is not None)


def _pattern(patterns: dict, module: str, default):
    """A module's own value: the pattern that is the module's path or the end of it, else the default."""
    for key, value in patterns.items():
        if module == key or module.endswith("." + key):
            return value
    return default


def read_adapter(path: str | Path) -> Entries:
    """An adapter directory's matrices with their scales (``lora_alpha / r``, or over its root where the configuration says so). What this framework
    has no place for -- other adapter kinds, trained biases, whole modules, embeddings -- is refused by name. The matrices keep the file's type here and are rounded
    to the weights' when the stacks are built, as the products read them."""
    path = Path(path)
    config, weights = (path / f for f in FILES)
    if not config.is_file() or not weights.is_file():
        raise AdapterError(f"{path}: an adapter directory holds {FILES[0]} and {FILES[1]}")
    try:
        cfg = json.loads(config.read_text())
    except (OSError, ValueError) as e:
        raise AdapterError(f"{config}: {e}")
    if not isinstance(cfg, dict) or str(cfg.get("peft_type", "LORA")).upper() != "LORA":
        raise AdapterError(f"{config}: not a LoRA adapter")
    if cfg.get("bias", "none") != "none" or cfg.get("modules_to_save"):
        raise AdapterError(f"{config}: trained biases and whole modules are not supported")
    for key in ("use_dora", "fan_in_fan_out", "lora_bias", "use_qalora", "trainable_token_indices", "alora_invocation_tokens", "layer_replication"):
        if cfg.get(key):
            raise AdapterError(f"{config}: {key} is not supported")
    init = cfg.get("init_lora_weights")
    if isinstance(init, str) and init.lower().startswith(REBASED):
        raise AdapterError(f"{config}: adapters that begin as {init} take a part of the model's weights into themselves; convert them to plain ones first")
    alpha, root = cfg.get("lora_alpha", 8), bool(cfg.get("use_rslora"))
    alphas = cfg.get("alpha_pattern") or {}
    if not isinstance(alphas, dict) or any(re.fullmatch(r"[\w.]+", k) is None for k in alphas):
        raise AdapterError(f"{config}: alpha_pattern takes module paths or ends of them, not expressions")
    found: dict[tuple[int, str], dict] = {}
    try:
        f = SafetensorsFile(weights)
    except (OSError, ValueError) as e:
        raise AdapterError(f"{weights}: {e}")
    for name in f.tensors:
        m = _NAME.search(name)
        if m is None or m.group(3) not in PROJECTIONS[m.group(2)]:
            raise AdapterError(f"{weights.name}: {name} changes none of the decoder's projections")
        layer, proj, side = int(m.group(1)), m.group(3), m.group(4)
        module = name[: name.index(".lora_")]
        entry = found.setdefault((layer, proj), {"module": module.removeprefix("base_model.model.")})
        if side in entry:
            raise AdapterError(f"{weights.name}: {name} is a second lora_{side} of layer {layer} {proj}")
        entry[side] = f.tensor(name).clone()
    entries: Entries = {}
    for (layer, proj), e in found.items():
        if "A" not in e or "B" not in e or e["A"].dim() != 2 or e["B"].dim() != 2 or e["A"].shape[0] != e["B"].shape[1] or e["A"].shape[0] == 0:
            raise AdapterError(f"{weights.name}: layer {layer} {proj} needs lora_A [r, in] and lora_B [out, r]")
        r = e["A"].shape[0]
        value = _pattern(alphas, e["module"], alpha)
        if not isinstance(value, (int, float)) or isinstance(value, bool) or not math.isfinite(value):
            raise AdapterError(f"{config}: lora_alpha must be a number")
        entries[layer, proj] = (e["A"], e["B"], float(value) / (math.sqrt(r) if root else r))
    if not entries:
        raise AdapterError(f"{weights.name}: holds no adapter matrices")
    return entries


def _one_part(entries: list, columns: list[int]) -> list:
    """Parts of a fused projection as one: ranks side by side, each part's B in its own columns (for parts that are not whole 64 columns)."""
    out = []
    for parts in entries:
        have = [(p, c) for p, c in zip(parts, range(len(columns))) if p is not None]
        if not have:
            out.append([None])
            continue
        a = torch.cat([p[0].float() for p, _ in have])
        b = torch.zeros(sum(columns), a.shape[0])
        at = 0
        for (pa, pb, scale), c in have:
            first = sum(columns[:c])
            b[first: first + columns[c], at: at + pa.shape[0]] = pb.float()
            at += pa.shape[0]
        out.append([(a, b, torch.cat([torch.full((p[0].shape[0],), float(p[2])) for p, _ in have]))])
    return out


def build_adapters(model, adapters: dict[str, Entries]) -> AdapterSet:
    """The stacks of a loaded decoder's layers. Refused where a layer's products are not the framework's plain BF16 ones on one GPU."""
    from ..models.decoder import DecoderModel, NoComm
    me, w, spec = type(model), model.w, model.spec
    if not all(getattr(me, f) is getattr(DecoderModel, f) for f in ("_attention", "_ffn", "hidden_states")) or spec.mla is not None:
        raise AdapterError(f"adapters are not available for {spec.arch}")
    if w.tp.size != 1 or type(model.comm) is not NoComm:
        raise AdapterError("adapters are not available with tensor parallelism")
    if w.embed.is_cuda and w.embed.dtype != torch.bfloat16:
        raise AdapterError("adapters need BF16 weights on a GPU")
    for i, name in enumerate(adapters):
        for (layer, proj), (a, b, _) in adapters[name].items():
            if layer >= spec.layers:
                raise AdapterError(f"adapter {name}: layer {layer} of a model of {spec.layers}")
            n, k = _shape(spec, w.layers[layer], proj)
            if n == 0:
                raise AdapterError(f"adapter {name}: layer {layer} has no plain {proj}")
            if a.shape[1] != k or b.shape[0] != n:
                raise AdapterError(f"adapter {name}: layer {layer} {proj} is [{n}, {k}], the adapter's [{b.shape[0]}, {a.shape[1]}]")
    layers = []
    try:
        for i, lw in enumerate(w.layers):
            stacks = LayerStacks()
            for field_, projs, weight in (("qkv", ("q_proj", "k_proj", "v_proj"), lw.wqkv), ("o", ("o_proj",), lw.wo),
                                          ("gu", ("gate_proj", "up_proj"), lw.wgu), ("down", ("down_proj",), lw.wdown)):
                entries = [[e.get((i, p)) for p in projs] for e in adapters.values()]
                if not any(p is not None for e in entries for p in e):
                    continue
                if not isinstance(weight, torch.Tensor):
                    raise AdapterError("adapters need BF16-resident weights")
                columns = [_shape(spec, lw, p)[0] for p in projs]
                interleave = field_ == "gu" and lw.wgu_interleaved
                if len(projs) > 1 and any(c % 64 for c in columns):
                    entries, columns, interleave = _one_part(entries, columns), [sum(columns)], False
                setattr(stacks, field_, lora_ops.pack_stack(entries, weight.shape[1], columns, weight.device, weight.dtype, interleave))
            layers.append(stacks)
    except lora_ops.KernelError as e:
        raise AdapterError(str(e))
    return AdapterSet(list(adapters), layers)


def _shape(spec: ModelSpec, lw, proj: str) -> tuple[int, int]:
    """(N, K) of a projection; N = 0 where the layer has none of its own (a mixture's experts, for instance)."""
    h = spec.hidden
    if proj == "q_proj":
        return spec.q_dim, h
    if proj in ("k_proj", "v_proj"):
        return spec.kv_dim, h
    if proj == "o_proj":
        return h, spec.q_dim
    if lw.router is not None or lw.wdown is None:
        return 0, 0
    f = lw.wdown.shape[1]
    return (h, f) if proj == "down_proj" else (f, h)
