"""Frequencies of rotary positions, also as checkpoints stretch them for contexts longer than they were trained on (the `rope_scaling` of a config.json, transformers
modeling_rope_utils' kinds): what lib.rotary and lib.rotary_kv_append take, in turns per position (inverse frequency / 2 pi) and in 64 bits."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch


KINDS = ("default", "linear", "yarn", "llama3")


def _number(scaling: dict, key: str, default: Optional[float] = None) -> float:
    v = scaling.get(key, default)
    if v is None:
        raise ValueError(f"rope_scaling of type {kind(scaling)!r} needs {key!r}")
    return float(v)


def kind(scaling: Optional[dict]) -> str:
    if not scaling:
        return "default"
    return str(scaling.get("rope_type") or scaling.get("type") or "default")


def frequencies(rot_dims: int, theta: float, scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float]:
    """(turns float64 [rot_dims / 2], the factor on cosine and sine).

    Pair i of rot_dims / 2 turns by theta^(-2i / rot_dims) radians per position. `scaling`:
    linear   every frequency divided by `factor`
    yarn     (Peng et al. 2023) pairs that make fewer than beta_slow turns over original_max_position_embeddings positions divided by `factor`, those that make more
             than beta_fast as they are, a straight ramp over the pairs between; cosine and sine times attention_factor, or 0.1 ln(factor) + 1
    llama3   wavelengths above original / low_freq_factor divided by `factor`, below original / high_freq_factor as they are, between them mixed by the turns made"""
    if rot_dims < 0 or rot_dims % 2:
        raise ValueError(f"an even number of rotated dimensions, not {rot_dims}")
    f = [float(theta) ** (-2.0 * i / rot_dims) for i in range(rot_dims // 2)]
    what, m = kind(scaling), 1.0
    if what == "linear":
        factor = _number(scaling, "factor")
        f = [x / factor for x in f]
    elif what == "yarn":
        factor, span = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        fast, slow = _number(scaling, "beta_fast", 32.0), _number(scaling, "beta_slow", 1.0)
        pair = lambda turns: rot_dims * math.log(span / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731  the pair that makes so many turns
        low, high = pair(fast), pair(slow)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rot_dims - 1)
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(rot_dims // 2)]
        f = [x / factor * r + x * (1.0 - r) for x, r in zip(f, ramp)]
        grown = lambda k: 0.1 * k * math.log(factor) + 1.0 if factor > 1.0 else 1.0  # noqa: E731
        if scaling.get("attention_factor") is not None:
            m = float(scaling["attention_factor"])
        elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
            m = grown(float(scaling["mscale"])) / grown(float(scaling["mscale_all_dim"]))
        else:
            m = grown(1.0)
    elif what == "llama3":
        factor, span = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings")
        slow, fast = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")

        def mixed(x):
            turns = span * x / (2 * math.pi)
            part = min(1.0, max(0.0, (turns - slow) / (fast - slow)))
            return x / factor * (1.0 - part) + x * part
        f = [mixed(x) for x in f]
    elif what != "default":
        raise NotImplementedError(f"rope_scaling of type {what!r} (built: {', '.join(KINDS[1:])})")
    return torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64, device=device), m
