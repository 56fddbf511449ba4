"""Loading a quantized checkpoint into the quantized Linear modules.

The reference keeps its quantization settings under ``quantization_config`` in the checkpoint's
``config.json`` (core/config.py:8-112) and loads by first swapping every ``nn.Linear`` of the model for an
empty quantized module (``from_linear(..., init_only=True)``, core/base.py:306-340) and then filling the
buffers by name from the checkpoint files (core/base.py:213-221).  The modules of this package keep the
reference's buffer names, shapes and dtypes, so the same two steps work on a reference-format checkpoint:

    cfg = QuantConfig.from_pretrained(path)
    replace_linears(model, cfg, dtype=torch.bfloat16)
    load_quantized_weights(model, path)

Only local directories and ``.safetensors`` files are read; nothing is downloaded.  FP8 checkpoints store
their weights as fp8-representable values in the model dtype; the modules cast them to fp8 once, on the
first forward, instead of on every forward (nn_models/modules/linear/linear_fp8.py:188).
"""
from __future__ import annotations

import json
import os
from dataclasses import dataclass, field
from typing import Iterable

import torch
from torch import nn

from .linear import FP8BlockGroupedLinear, FP8BlockLinear, SqW8A8BBF16OBF16PerChannel, SqW8A8GroupedLinear, method_to_linear


@dataclass
class QuantConfig:
    """Field names and defaults of the reference's QuantConfig (core/config.py:9-20), and one for block-scaled checkpoints."""
    quant_method: str = "awq"          # "awq" | "sq" | "fp8_static_quant" | "fp8_dynamic_quant"
    zero_point: bool = False
    q_group_size: int = 0
    w_bit: int = 8
    version: str = "gemm"
    modules_to_not_convert: list = field(default_factory=lambda: ["lm_head"])
    fp8_static_quant: bool = False
    kv_cache_quant_layers: list = field(default_factory=list)
    per_tensor: bool = True
    skip_whole_names: bool = False     # modules_to_not_convert lists whole parts of names (published fp8 checkpoints), not any piece of one

    @classmethod
    def from_dict(cls, d: dict | None = None) -> "QuantConfig":
        cfg = cls(**d) if d else cls()
        cfg.version = cfg.version.lower()
        return cfg

    @classmethod
    def from_transformers_dict(cls, d: dict) -> "QuantConfig":
        """The key names used inside config.json (core/config.py:88-112): group_size, bits.  Block-scaled fp8 checkpoints as published have names of their
        own, quant_method "fp8" with a weight_block_size: of 128 x 128 with dynamic scales of the activations, they are this package's
        "fp8_dynamic_quant" with groups of 128; of any other kind they keep their quant_method, which replace_linears refuses."""
        if d.get("quant_method") == "fp8" and list(d.get("weight_block_size") or ()) == [128, 128] and d.get("activation_scheme", "dynamic") == "dynamic":
            d = {**d, "quant_method": "fp8_dynamic_quant", "group_size": 128, "bits": 8, "skip_whole_names": True}
        known = {"quant_method": "quant_method", "zero_point": "zero_point", "group_size": "q_group_size",
                 "bits": "w_bit", "fp8_static_quant": "fp8_static_quant",
                 "kv_cache_quant_layers": "kv_cache_quant_layers",
                 "modules_to_not_convert": "modules_to_not_convert", "per_tensor": "per_tensor", "skip_whole_names": "skip_whole_names"}
        kwargs = {ours: d[theirs] for theirs, ours in known.items() if d.get(theirs) is not None}
        return cls.from_dict(kwargs)

    @classmethod
    def from_pretrained(cls, save_dir: str) -> "QuantConfig":
        path = os.path.join(save_dir, "config.json")
        if not os.path.isfile(path):
            raise FileNotFoundError(f"{path}: only local checkpoint directories are supported")
        with open(path, "r", encoding="utf-8") as f:
            loaded = json.load(f)
        q = loaded.get("quantization_config")
        return cls.from_transformers_dict(q) if q else cls()

    def to_transformers_dict(self) -> dict:
        d = {"quant_method": self.quant_method, "zero_point": self.zero_point, "group_size": self.q_group_size,
             "bits": self.w_bit, "fp8_static_quant": self.fp8_static_quant,
             "kv_cache_quant_layers": self.kv_cache_quant_layers,
             "modules_to_not_convert": self.modules_to_not_convert, "per_tensor": self.per_tensor}
        return {**d, "skip_whole_names": True} if self.skip_whole_names else d


def _set_submodule(root: nn.Module, name: str, new: nn.Module) -> None:
    parent = root
    parts = name.split(".")
    for p in parts[:-1]:
        parent = parent[int(p)] if p.isdigit() and not hasattr(parent, p) else getattr(parent, p)
    setattr(parent, parts[-1], new)


def replace_linears(model: nn.Module, cfg: QuantConfig, dtype=torch.bfloat16) -> list[str]:
    """Swap every nn.Linear whose name contains none of ``cfg.modules_to_not_convert`` for an empty quantized
    module of the configured kind (buffers allocated, not filled).  -> the names that were replaced.

    ``quant_method == "sq"`` with ``per_tensor == False`` selects the per-token x per-channel SmoothQuant module,
    which the reference declares but does not implement; ``quant_method == "fp8_dynamic_quant"`` with ``q_group_size == 128`` the block-scaled FP8
    module, whose weight is stored in e4m3fn with a scale per 128 x 128 block (the reference's FP8 modules refuse any group size but 0).  With
    ``skip_whole_names`` a name is skipped only where whole parts of it are listed ("mlp.gate" is no part of "mlp.gate_proj").  The modules of a list of experts are replaced one by
    one; the from_linears of FP8BlockGroupedLinear and SqW8A8GroupedLinear joins them once they are filled."""
    if cfg.quant_method not in method_to_linear:
        raise RuntimeError(f"quant_method {cfg.quant_method!r} is not supported: {sorted(method_to_linear)}, or \"fp8\" with a weight_block_size of 128 x 128 "
                           "and dynamic activation scales")
    kind = method_to_linear[cfg.quant_method]
    if cfg.quant_method == "sq" and not cfg.per_tensor:
        kind = SqW8A8BBF16OBF16PerChannel
    if cfg.quant_method == "fp8_dynamic_quant" and cfg.q_group_size == 128:
        kind = FP8BlockLinear
    skip = cfg.modules_to_not_convert or []
    skipped = (lambda n: any(f".{key}." in f".{n}." for key in skip)) if cfg.skip_whole_names else (lambda n: any(key in n for key in skip))
    targets = [(n, m) for n, m in model.named_modules()
               if isinstance(m, nn.Linear) and n and not skipped(n)]
    for name, lin in targets:
        q = kind.from_linear(lin, cfg.w_bit, cfg.q_group_size, True, dtype=dtype, per_tensor=cfg.per_tensor)
        _set_submodule(model, name, q)
    return [n for n, _ in targets]


def _checkpoint_files(path: str) -> list[str]:
    if os.path.isfile(path):
        return [path]
    index = os.path.join(path, "model.safetensors.index.json")
    if os.path.isfile(index):
        with open(index, "r", encoding="utf-8") as f:
            names = sorted(set(json.load(f)["weight_map"].values()))
        return [os.path.join(path, n) for n in names]
    files = sorted(os.path.join(path, f) for f in os.listdir(path) if f.endswith(".safetensors"))
    if not files:
        raise FileNotFoundError(f"no .safetensors files under {path}")
    return files


def load_quantized_weights(model: nn.Module, path: str, device=None) -> tuple[list[str], list[str]]:
    """Fill parameters and buffers by name from the ``.safetensors`` file(s) at ``path`` (a file, a directory,
    or a directory with a ``model.safetensors.index.json``).  Shapes and dtypes must match what the modules
    allocated (scalars may come as 0-dim or 1-element tensors).  Floating-point values are converted; what becomes 8 bits must be such values already
    (codes that are stored in a wider type), since an unquantized weight would lose most of its bits unseen.  A directory that holds a block-scaled
    module's weight must hold its scales too, which may be named ``weight_scale_inv`` (the factor of the codes all the same).  Codes with
    scales are refused for an nn.Linear.  -> (missing names, unexpected names)."""
    from safetensors import safe_open

    own = dict(model.named_parameters())
    own.update(dict(model.named_buffers()))
    modules = dict(model.named_modules())
    block_scaled = (FP8BlockLinear, FP8BlockGroupedLinear)
    seen, unexpected, plain = set(), [], []
    for file in _checkpoint_files(path):
        with safe_open(file, framework="pt", device="cpu") as f:
            for key in f.keys():
                stored, (prefix, _, last) = key, key.rpartition(".")
                owner = modules.get(prefix)
                if isinstance(owner, block_scaled) and last == "weight_scale_inv":
                    key = key.removesuffix("_inv")
                dst = own.get(key)
                if dst is None:
                    unexpected.append(stored)
                    continue
                src = f.get_tensor(stored)
                if src.numel() == dst.numel() and src.shape != dst.shape and dst.numel() == 1:
                    src = src.reshape(dst.shape)
                if src.shape != dst.shape:
                    raise RuntimeError(f"{key}: checkpoint shape {tuple(src.shape)} != module shape {tuple(dst.shape)}")
                if src.dtype != dst.dtype and not (src.is_floating_point() and dst.is_floating_point()):
                    raise RuntimeError(f"{key}: checkpoint dtype {src.dtype} != module dtype {dst.dtype}")
                if type(owner) is nn.Linear and src.dtype.itemsize == 1 and src.is_floating_point():
                    plain.append(key)
                cast = src.to(dst.dtype)
                if dst.dtype.itemsize == 1 and src.dtype != dst.dtype and not torch.equal(cast.float(), src.float()):
                    raise RuntimeError(f"{key}: values in {src.dtype} that are no {dst.dtype} codes; an unquantized weight must be quantized first")
                with torch.no_grad():
                    dst.copy_(cast)
                seen.add(key)
    for key in plain:
        if f"{key}_scale" in unexpected or f"{key}_scale_inv" in unexpected:
            raise RuntimeError(f"{key}: the checkpoint holds codes and scales for a module that is not quantized")
    for name, m in modules.items():
        weight, scale = (f"{name}.{t}" if name else t for t in ("weight", "weight_scale"))
        if not os.path.isfile(path) and isinstance(m, block_scaled) and weight in seen and scale not in seen:
            raise RuntimeError(f"{scale}: the checkpoint holds the codes of {weight} and no scales for them")
    for m in model.modules():   # cached fp8 casts of weights that were just overwritten
        if hasattr(m, "invalidate_cache"):
            m.invalidate_cache()
    if device is not None:
        model.to(device)
    return sorted(k for k in own if k not in seen), unexpected


def named_quantized_linears(model: nn.Module) -> Iterable[tuple[str, nn.Module]]:
    kinds = tuple(set(method_to_linear.values()) | {SqW8A8BBF16OBF16PerChannel, SqW8A8GroupedLinear, FP8BlockLinear, FP8BlockGroupedLinear})
    return ((n, m) for n, m in model.named_modules() if isinstance(m, kinds))
