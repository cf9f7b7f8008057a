"""Low-rank adapters from a folder: adapter_config.json ("r", "lora_alpha") and adapter_model.safetensors with a pair of matrices
per projection, named ``...layers.<i>.self_attn.q_proj.lora_A.weight`` [rank, in] and ``...lora_B.weight`` [out, rank]."""
from __future__ import annotations

import json
import os
import re
from typing import Dict, List, Optional, Tuple

import torch

from .safetensors_io import SafetensorsFile, write_safetensors

# where a published name goes: (projection of the part, place among what is stacked in it, parts stacked)
PLACES = {"self_attn.q_proj": ("w_qkv", 0, 3), "self_attn.k_proj": ("w_qkv", 1, 3), "self_attn.v_proj": ("w_qkv", 2, 3),
          "self_attn.o_proj": ("w_o", 0, 1), "mlp.gate_proj": ("w_gate_up", 0, 2), "mlp.up_proj": ("w_gate_up", 1, 2),
          "mlp.down_proj": ("w_down", 0, 1)}
_NAME = re.compile(r"(?:.*\.)?layers\.(\d+)\.(\w+\.\w+)\.lora_([AB])(?:\.default)?\.weight$")


def read_adapter(folder: str) -> Tuple[Dict[Tuple[int, str], List[Optional[Tuple[torch.Tensor, torch.Tensor]]]], float]:
    """({(layer, projection): (down, up) or None for every part stacked in it}, scale)."""
    with open(os.path.join(folder, "adapter_config.json")) as f:
        config = json.load(f)
    rank, alpha = int(config["r"]), float(config.get("lora_alpha", config["r"]))
    if rank < 1:
        raise ValueError(f"{folder}: rank {rank}")
    if config.get("use_dora") or config.get("rank_pattern") or config.get("alpha_pattern"):
        raise ValueError(f"{folder}: adapters with magnitudes or a rank of their own per projection are not supported")
    scale = alpha / rank ** 0.5 if config.get("use_rslora") else alpha / rank
    halves: Dict[Tuple[int, str], Dict[str, torch.Tensor]] = {}
    unexpected = []
    with SafetensorsFile(os.path.join(folder, "adapter_model.safetensors")) as f:
        for name in f.names():
            m = _NAME.match(name)
            if m is None or m.group(2) not in PLACES:
                unexpected.append(name)
                continue
            halves.setdefault((int(m.group(1)), m.group(2)), {})[m.group(3)] = f.tensor(name)
    if unexpected:
        raise ValueError(f"{folder}: tensors that no projection takes: {', '.join(sorted(unexpected)[:5])}")
    pairs: Dict[Tuple[int, str], List] = {}
    for (layer, published), half in halves.items():
        if set(half) != {"A", "B"}:
            raise ValueError(f"{folder}: layer {layer}, {published}: one matrix of the pair is missing")
        name, place, stacked = PLACES[published]
        pairs.setdefault((layer, name), [None] * stacked)[place] = (half["A"], half["B"])
    return pairs, scale


def write_random_adapter(config, seed: int, folder: str, rank: int = 8, alpha: float = 16.0, std: float = 0.02) -> None:
    """A folder with a random adapter for every projection of a Llama configuration (a ``LlamaConfig``), for tests and measurements."""
    g = torch.Generator().manual_seed(seed)
    D, I, hd = config.hidden_size, config.intermediate_size, config.head_dim
    sizes = {"self_attn.q_proj": (D, config.num_attention_heads * hd), "self_attn.k_proj": (D, config.num_key_value_heads * hd),
             "self_attn.v_proj": (D, config.num_key_value_heads * hd), "self_attn.o_proj": (config.num_attention_heads * hd, D),
             "mlp.gate_proj": (D, I), "mlp.up_proj": (D, I), "mlp.down_proj": (I, D)}
    tensors = []
    for layer in range(config.num_hidden_layers):
        for name, (k, n) in sizes.items():
            at = f"base_model.model.model.layers.{layer}.{name}"
            tensors.append((f"{at}.lora_A.weight", (torch.randn(rank, k, generator=g) * std).to(torch.bfloat16)))
            tensors.append((f"{at}.lora_B.weight", (torch.randn(n, rank, generator=g) * std).to(torch.bfloat16)))
    os.makedirs(folder, exist_ok=True)
    write_safetensors(os.path.join(folder, "adapter_model.safetensors"), tensors)
    with open(os.path.join(folder, "adapter_config.json"), "w") as f:
        json.dump({"r": rank, "lora_alpha": alpha, "target_modules": [n.split(".")[1] for n in sizes]}, f)
