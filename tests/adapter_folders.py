"""Adapter folders for the tiny test models, and the same models with an adapter merged into their weights."""

import json
import os
import tempfile

import numpy as np
import torch

from reflex_b200.weights import write_safetensors

ROLES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj",
         "mlp.down_proj")


def adapter_folder(cfg, rank, seed, roles=ROLES, layers=None, alpha=None, size=0.3, **more):
    """(folder, {tensor name: (A, B)}): random A and B, W's size times `size` a product."""
    rng = torch.Generator().manual_seed(seed)
    H, I, d = cfg["hidden_size"], cfg["intermediate_size"], cfg["head_dim"]
    q, kv = cfg["num_attention_heads"] * d, cfg["num_key_value_heads"] * d
    shape = {"self_attn.q_proj": (q, H), "self_attn.k_proj": (kv, H), "self_attn.v_proj": (kv, H), "self_attn.o_proj": (H, q),
             "mlp.gate_proj": (I, H), "mlp.up_proj": (I, H), "mlp.down_proj": (H, I)}
    pairs, tensors = {}, []
    for l in range(cfg["num_hidden_layers"]) if layers is None else layers:
        for role in roles:
            out, width = shape[role]
            a = torch.randn(rank, width, generator=rng) * 0.02
            b = torch.randn(out, rank, generator=rng) * size * rank ** -0.5
            module = f"model.layers.{l}.{role}"
            pairs[module + ".weight"] = (a, b)
            tensors += [(f"base_model.model.{module}.lora_A.weight", a), (f"base_model.model.{module}.lora_B.weight", b)]
    folder = tempfile.mkdtemp(prefix="rfx_adapter_")
    write_safetensors(os.path.join(folder, "adapter_model.safetensors"), tensors)
    with open(os.path.join(folder, "adapter_config.json"), "w") as f:
        json.dump(dict(r=rank, lora_alpha=rank if alpha is None else alpha, **more), f)
    return folder, pairs


def merged(weights, pairs, scale=1.0):
    """The plain model's weights with an adapter added into them."""
    out = dict(weights)
    for name, (a, b) in pairs.items():
        out[name] = (weights[name].astype(np.float64) + scale * (b.double() @ a.double()).numpy()).astype(np.float32)
    return out
