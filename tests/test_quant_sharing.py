"""Quantising a model changes its parts, which every engine of the model runs: what is refused, and that a refused model is as it was. No GPU."""
import copy
import gc
import weakref

import pytest
import torch

import tiny
from rllm_b200.config import config_from_dict
from rllm_b200.engine import factory, step
from rllm_b200.engine.factory import set_kv_quant, set_weight_quant
from rllm_b200.kernels import quant
from rllm_b200.parts import KV4CacheSpec, Part


class AnEngine:
    pass


def model_of(cfg):
    arch, c = config_from_dict(cfg)
    return arch.build(c)


def bound():
    """A Llama with weights, whose matrices are quantised without a GPU."""
    m = model_of(tiny.TINY["D"][0])
    for p in m.parts():
        for q in p.params():
            setattr(p, q.attr, torch.zeros(q.shape))
    return m


@pytest.fixture
def on_cpu(monkeypatch):
    import contextlib
    made = []

    def make(w):
        made.append(w)
        return quant.Int8Matrix(torch.zeros(w.shape[0], -(-w.shape[1] // 16) * 16, dtype=torch.int8), torch.zeros(w.shape[0]), w.shape[1])
    monkeypatch.setattr(quant, "quantize_matrix", make)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    return made


def kinds(m):
    return [type(s) for s in m.cache_specs()]


def test_a_model_that_an_engine_runs_is_not_changed(on_cpu):
    m = bound()
    e = AnEngine()
    e.me = e                                               # (as an engine and its captured steps do)
    step._engines[m] = weakref.WeakSet([e])
    twin = copy.deepcopy(m)                                # parts of its own, which no engine runs
    before = kinds(m), [getattr(p, n) for p in m.parts() for n in p.int8_params]
    with pytest.raises(ValueError, match="another engine"):
        set_kv_quant(m, "int4")
    with pytest.raises(ValueError, match="another engine"):
        set_weight_quant(m, "int8")
    set_kv_quant(m, "none")
    set_weight_quant(m, "none")
    after = kinds(m), [getattr(p, n) for p in m.parts() for n in p.int8_params]
    assert before[0] == after[0] and all(a is b for a, b in zip(before[1], after[1])) and not on_cpu
    set_kv_quant(twin, "int4")
    assert all(k is KV4CacheSpec for k in kinds(twin)) and kinds(m) == before[0]
    del e                                                  # nothing runs it any more
    set_kv_quant(m, "int4")
    set_weight_quant(m, "int8")
    assert all(k is KV4CacheSpec for k in kinds(m)) and on_cpu
    n = len(on_cpu)
    step._engines[m].add(e := AnEngine())
    set_kv_quant(m, "int4")                                # a second engine of the same kind
    set_weight_quant(m, "int8")
    assert len(on_cpu) == n and e in step._engines[m]


def test_a_quantised_model_does_not_turn_back_in_silence(on_cpu):
    m = bound()
    set_kv_quant(m, "int4")
    set_weight_quant(m, "int8")
    with pytest.raises(ValueError, match="load it again"):
        set_kv_quant(m, "none")
    with pytest.raises(ValueError, match="load it again"):
        set_weight_quant(m, "none")


def test_a_refused_model_is_as_it_was(on_cpu, monkeypatch):
    m = bound()
    last = [p for p in m.parts() if hasattr(p, "use_kv4")][-1]
    position = last.position
    last.position = Part()                                 # the last layer's position encoding writes the cache itself
    before = kinds(m)
    with pytest.raises(ValueError, match="does not write"):
        set_kv_quant(m, "int4")
    assert kinds(m) == before and KV4CacheSpec not in before
    last.position = position

    def refuse(*a):
        raise ValueError("refused")
    monkeypatch.setattr(factory, "set_weight_quant", refuse)          # an engine whose weights are refused leaves no layer at 4 bits
    with pytest.raises(ValueError, match="refused"):
        factory.make_engine(m, "bfloat16", kv_quant="int4", weight_quant="int8")
    assert kinds(m) == before


def test_an_engine_is_known_while_it_lives():
    from rllm_b200.engine.step import Engine, any_engine

    class NoModel:
        vocab_size = 8

    class NoBackend:
        fast, device = False, torch.device("cpu")

    m = NoModel()
    assert not any_engine(m)
    a, b = (Engine(m, NoBackend(), None, use_graphs=False) for _ in range(2))
    assert any_engine(m) and len(step._engines[m]) == 2
    del a, b
    gc.collect()
    assert not any_engine(m)


def test_a_model_that_would_be_quantised_in_part_is_refused(on_cpu):
    """Livovik's shared expert is a SwiGLU like Llama's; its attention and its routed experts have matrices of their own kinds."""
    from livovik_tiny import LA
    m = model_of(LA)
    with pytest.raises(ValueError, match="SinkGQAttention.*cannot be held in 8 bits"):
        set_weight_quant(m, "int8")
    assert not on_cpu
