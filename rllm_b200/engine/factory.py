"""From a model folder (or a configuration and a seed) to an `Engine`: configuration ->
registry -> parts -> weights -> cache pool -> step function. The counterpart of the
reference's `load_and_run_single_gpu` (src/engine/loader.rs:229-398)."""
from __future__ import annotations

import torch

from ..cache import CacheManager, pages_for
from ..config import config_from_dict, load_config
from ..kernels.backend import Backend
from ..parts.base import KV4CacheSpec, cache_kind_of
from ..weights import init_random_weights, load_weights
from .step import Engine, any_engine

_DTYPES = {"bfloat16": torch.bfloat16, "bf16": torch.bfloat16,
           "float32": torch.float32, "fp32": torch.float32, "f32": torch.float32}


def parse_dtype(name) -> torch.dtype:
    if isinstance(name, torch.dtype):
        return name
    try:
        return _DTYPES[str(name).lower()]
    except KeyError:
        raise ValueError(f"dtype must be one of {sorted(_DTYPES)}, got {name!r}") from None


KV_QUANT = ("none", "int4")
WEIGHT_QUANT = ("none", "int8")


def _may_change(model, what: str, asked: str, has: str) -> bool:
    """Is the model to be changed from the form that it `has` to the one asked for? Its parts are what every engine of it runs, with their captured
    steps: the form is chosen before the first, and never taken back."""
    if asked == has:
        return False
    if has != "none":
        raise ValueError(f"{what} {asked!r}: this model has been given {what} {has!r}, which cannot be taken back; load it again")
    if any_engine(model):
        raise ValueError(f"{what} {asked!r}: another engine runs this model with {what} 'none'; load it again for this one")
    return True


def set_kv_quant(model, kv_quant: str) -> list:
    """"int4": every layer's keys and values are held in 4 bits (`KV4CacheSpec`); a model with another paged cache is refused and left as it
    was, and so is one that an engine runs otherwise. Before the cache is made. Returns the parts that were changed."""
    if kv_quant not in KV_QUANT:
        raise ValueError(f"kv_quant must be one of {KV_QUANT}, got {kv_quant!r}")
    able = [p for p in model.parts() if hasattr(p, "use_kv4")]
    if not _may_change(model, "kv_quant", kv_quant, "int4" if any(getattr(p, "kv4", False) for p in able) else "none"):
        return []
    specs = [s for s in model.cache_specs() if s is not None and cache_kind_of(s).paged]
    if not able:
        raise ValueError(f"kv_quant {kv_quant!r}: this model has no cache of keys and values that can be held in 4 bits"
                         + (f" (it has {sorted({type(s).__name__ for s in specs})})" if specs else ""))
    try:
        for p in able:
            p.use_kv4()
        left = sorted({type(s).__name__ for s in model.cache_specs()
                       if s is not None and cache_kind_of(s).paged and not isinstance(s, KV4CacheSpec)})
        if left:
            raise ValueError(f"kv_quant {kv_quant!r}: layers with {left} cannot be held in 4 bits")
    except ValueError:
        for p in able:
            p.kv4 = False
        raise
    return able


def set_weight_quant(model, weight_quant: str) -> None:
    """"int8": the matrices that the parts declare (`Part.int8_params`) are held in 8 bits with a scale per output channel, and their
    inputs are quantised per token. Embedding and output head stay as they are; a model whose layers have other matrices is refused, and so is one
    that an engine runs otherwise. After the weights are bound."""
    if weight_quant not in WEIGHT_QUANT:
        raise ValueError(f"weight_quant must be one of {WEIGHT_QUANT}, got {weight_quant!r}")
    from ..kernels import quant
    held = [(p, n) for p in model.parts() for n in p.int8_params]
    has = any(isinstance(getattr(p, n), quant.Int8Matrix) for p, n in held)
    if not _may_change(model, "weight_quant", weight_quant, "int8" if has else "none"):
        return
    if not held:
        raise ValueError(f"weight_quant {weight_quant!r}: no part of this model has matrices that can be held in 8 bits")
    left = sorted({f"{type(p).__name__}.{q.attr}" for b in model.blocks for p in b.walk() for q in p.params()
                   if len(q.shape) > 1 and q.role == "matrix" and q.attr not in p.int8_params})
    if left:
        raise ValueError(f"weight_quant {weight_quant!r}: {', '.join(left)} cannot be held in 8 bits")
    for p, name in held:
        w = getattr(p, name)
        with torch.cuda.device(w.device):
            setattr(p, name, quant.quantize_matrix(w))
            del w
            torch.cuda.empty_cache()           # its memory goes back to the device, before the next one's codes are cut out of it


def default_num_pages(model, page_size: int, dtype: torch.dtype, device, weights_bytes: int = 0,
                      fraction: float = 0.75) -> int:
    """Pages that fit in `fraction` of the free device memory (the reference takes 75 % of
    what is left after the weights, src/model/config.rs:1195-1226, clamped there to
    [256, 8192] blocks; here only a floor is kept). What torch keeps of freed tensors is free too."""
    free = torch.cuda.mem_get_info(device)[0] + torch.cuda.memory_reserved(device) - torch.cuda.memory_allocated(device)
    per_page = CacheManager.bytes_per_page(model.cache_specs(), page_size, dtype)
    if per_page == 0:
        return 0
    return max(16, int(free * fraction) // per_page)


def make_engine(model, dtype, device="cuda:0", page_size: int = 16, num_pages: int | None = None,
                max_tokens: int | None = None, max_requests: int = 256, kv_quant: str = "none",
                weight_quant: str = "none") -> Engine:
    """`model` must already hold its weights on `device`."""
    dtype = parse_dtype(dtype)
    changed = set_kv_quant(model, kv_quant)
    try:
        set_weight_quant(model, weight_quant)
    except ValueError:
        for p in changed:
            p.kv4 = False
        raise
    backend = Backend(dtype, device)
    if num_pages is None:
        if max_tokens is not None:
            num_pages = pages_for(max_tokens, page_size)
        else:
            num_pages = default_num_pages(model, page_size, dtype, device)
    cache = CacheManager(model.cache_specs(), page_size, num_pages, max_requests, dtype, device)
    from ..kernels import profile
    if profile.enabled():
        # per-operation timing: every backend call bracketed by events, no graph replays
        return Engine(model, profile.OpProfile(backend), cache, use_graphs=False)
    return Engine(model, backend, cache)


def load_engine(model_dir: str, dtype="bfloat16", device="cuda:0", **kw) -> Engine:
    dtype = parse_dtype(dtype)
    arch, cfg = load_config(model_dir)
    model = arch.build(cfg)
    load_weights(model, model_dir, dtype, device)
    return make_engine(model, dtype, device, **kw)


def random_engine(config: dict, seed: int, dtype="bfloat16", device="cuda:0", std: float = 0.02,
                  norm_std: float = 0.0, **kw) -> Engine:
    dtype = parse_dtype(dtype)
    arch, cfg = config_from_dict(config)
    model = arch.build(cfg)
    init_random_weights(model, seed, dtype, device, std, norm_std)
    return make_engine(model, dtype, device, **kw)
