"""Engines that share a model, and what quantised weights leave to the cache."""
import gc

import pytest
import torch

import plain_llama as P
import tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_an_engine_with_captured_steps_keeps_its_weights(tmp_path):
    from rllm_b200.engine import Entry, load_engine
    from rllm_b200.engine.factory import make_engine
    d = tiny.make_model_dir(tmp_path, "D")
    toks = tiny.random_prompt(40, P.read_model_dir(d)[0]["vocab_size"], 3)
    a = load_engine(d, device=DEV, num_pages=16)
    a.step([Entry("a", toks, [39])])
    x = a.step([Entry("a", [5], [0])]).clone()
    assert a.graph_steps > 0
    for kw in ({"weight_quant": "int8"}, {"kv_quant": "int4"}, {"kv_quant": "int4", "weight_quant": "int8"}):
        with pytest.raises(ValueError, match="another engine"):
            make_engine(a.model, "bfloat16", device=DEV, num_pages=16, **kw)
    b = make_engine(a.model, "bfloat16", device=DEV, num_pages=16)               # in the same form it may
    b.step([Entry("a", toks, [39])])
    assert torch.equal(b.step([Entry("a", [5], [0])]), x)
    a.end(["a"])
    a.step([Entry("a", toks, [39])])
    assert torch.equal(a.step([Entry("a", [5], [0])]), x)
    model = a.model
    del a, b
    c = make_engine(model, "bfloat16", device=DEV, num_pages=16, kv_quant="int4", weight_quant="int8")
    assert torch.isfinite(c.step([Entry("a", toks, [39])])).all()


def test_the_cache_gets_the_memory_that_quantised_weights_leave():
    """`default_num_pages` behind `set_weight_quant`: of what the device has free, to which the matrices' other half belongs then."""
    from rllm_b200.config import config_from_dict
    from rllm_b200.engine.factory import default_num_pages, set_weight_quant
    from rllm_b200.cache import CacheManager
    from rllm_b200.weights import init_random_weights
    cfg = dict(tiny.TINY["D"][0], hidden_size=2048, intermediate_size=16384, num_attention_heads=16, num_key_value_heads=8, head_dim=64,
               num_hidden_layers=8)
    arch, c = config_from_dict(cfg)
    m = arch.build(c)
    init_random_weights(m, 1, torch.bfloat16, DEV)
    gc.collect()
    torch.cuda.empty_cache()
    held = [getattr(p, n) for p in m.parts() for n in p.int8_params]
    saved = sum(w.numel() for w in held)                   # bfloat16 to 8 bits: a byte a number
    del held
    per_page = CacheManager.bytes_per_page(m.cache_specs(), 16, torch.bfloat16)
    before = default_num_pages(m, 16, torch.bfloat16, DEV)
    set_weight_quant(m, "int8")
    after = default_num_pages(m, 16, torch.bfloat16, DEV)
    # three quarters of what is free, less the scales
    assert saved > 8e8 and after - before >= 0.75 * 0.9 * saved / per_page, (after - before, 0.75 * saved / per_page)
