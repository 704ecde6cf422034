"""Model registry: a configuration's `architecture` names the class that reads it.

A model class provides
    from_config(config, weights, device, dtype)   weights: checkpoint.Weights, or None for random ones
and its instances what the engine drives:
    device, vocab, num_layers, page_size (preferred), tau, seed
    make_caches(num_pages, page_size, max_len)     the step's cache, whatever the model keeps per token
    make_prefix(max_len) / None                    scratch for the prefilling entries' cached tokens, if it wants one
    step(caches, inp, ids, cached_lens, block_table, num_decoding, prefix, asks=) -> StepOutput
    logits(hidden)                                 fp32 or bf16 logits of normed rows
A class whose projections take low-rank adapters has make_adapters(slots, rank), which gives it empty slots, and `adapters`, a dict of
ops.Adapters per layer (None before).  A class with `stateful = True` keeps a state per request beside the pages: its make_caches takes slots=, the number of state
slots, and its step slots=, int32 [entries], the slot of every entry (-1: padding).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import kernels as K
from .. import ops

MODELS: dict[str, type] = {}


@dataclass
class StepOutput:
    tokens: torch.Tensor  # int64 [entries]: the sampled next token of every entry
    hidden: torch.Tensor  # [rows, width]: the final normed state of every packed row of the step


@dataclass
class Asks:
    """What a step's requests bring with them."""

    adapters: torch.Tensor | None = None  # int32 [rows]: every row's adapter slot, -1: none
    draw: ops.Draw | None = None  # how the entries' tokens are drawn; None: the model's tau and seed for all
    rules: ops.Rules | None = None


def plan_of(model, asks: Asks | None) -> ops.AdapterPlan | None:
    """The step's rows by adapter, for all its projections."""
    if asks is None or asks.adapters is None:
        return None
    if model.adapters is None:
        raise ValueError("rows with adapters, but the model has no slots for them (make_adapters)")
    return ops.plan_adapters(asks.adapters, next(iter(model.adapters[0].values())).slots)


def adapted(x: torch.Tensor, weight: torch.Tensor, adapters: ops.Adapters | None, plan: ops.AdapterPlan | None) -> torch.Tensor:
    """The shared projection of x, and every row's adapter beside it."""
    y = K.linear(x, weight)
    return y if plan is None or adapters is None else ops.add_adapters(y, x, adapters, plan)


def next_tokens(model, hidden: torch.Tensor, asks: Asks | None) -> torch.Tensor:
    """The next token of every entry from its last normed row: int64 [entries]."""
    logits = model.logits(hidden)
    if asks is None or asks.draw is None:
        return K.sample(logits, model.tau, model.seed).view(-1)
    return ops.choose_tokens(logits, asks.draw, asks.rules, append=asks.rules is not None and asks.rules.history is not None)[0]


def register(architecture: str):
    def add(cls):
        MODELS[architecture] = cls
        return cls

    return add


def load_all() -> dict[str, type]:
    """Import every model module (each registers itself)."""
    from .. import scaffold  # noqa: F401  (registers itself)
    from . import biranex, radivik  # noqa: F401

    return MODELS


def model_class(config: dict) -> type:
    load_all()
    name = config.get("architecture")
    if name not in MODELS:
        raise ValueError(f"unknown architecture {name!r}; known: {', '.join(sorted(MODELS))}")
    return MODELS[name]


def load_model(folder: str, device="cuda", dtype: torch.dtype = torch.bfloat16, random_weights: bool = False):
    """The model of a folder (config.json + safetensors).  random_weights: from the configuration alone."""
    from .. import checkpoint

    config = checkpoint.read_config(folder)
    weights = None if random_weights else checkpoint.Weights.open(folder)
    return model_class(config).from_config(config, weights, torch.device(device), dtype)
