"""Quantised serving without a GPU: which models and sizes take it, what the cache costs, what the command line and the kernels'
faces refuse."""
import pytest
import torch

import plain_quant as Q
import tiny
from rllm_b200 import cli
from rllm_b200.cache import CacheManager
from rllm_b200.config import config_from_dict
from rllm_b200.engine.factory import set_kv_quant, set_weight_quant
from rllm_b200.kernels import ops, quant
from rllm_b200.parts import KV4CacheSpec, KVCacheSpec, cache_kind_of
from zukotar_tiny import ZA


def model_of(cfg):
    arch, c = config_from_dict(cfg)
    return arch.build(c)


def test_the_cache_in_4_bits_is_a_kind_of_its_own():
    spec = KV4CacheSpec(8, 128, window=100)
    kind = cache_kind_of(spec)
    assert kind.paged and kind.window(spec) == 100
    t = kind.allocate(spec, 3, 16, torch.bfloat16, "cpu")
    assert {n: (tuple(x.shape), x.dtype) for n, x in t.items()} == {
        "k4": ((3, 8, 16, 64), torch.uint8), "v4": ((3, 8, 16, 64), torch.uint8),
        "ks": ((3, 8, 16, 4), torch.bfloat16), "vs": ((3, 8, 16, 4), torch.bfloat16)}
    assert 3 * kind.page_bytes(spec, 16, torch.bfloat16) == sum(x.nbytes for x in t.values())
    full = cache_kind_of(KVCacheSpec(8, 128)).page_bytes(KVCacheSpec(8, 128), 16, torch.bfloat16)
    assert full * 9 == kind.page_bytes(spec, 16, torch.bfloat16) * 32           # 4.5 bits a number for 16


@pytest.mark.parametrize("name", ["D", "E", "F"])
def test_a_model_that_takes_it(name):
    m = model_of(tiny.TINY[name][0])
    before = m.cache_specs()
    set_kv_quant(m, "none")
    assert m.cache_specs() == before
    set_kv_quant(m, "int4")
    assert [(type(s), s.kv_heads, s.head_dim, s.window) for s in m.cache_specs()] == \
        [(KV4CacheSpec, s.kv_heads, s.head_dim, s.window) for s in before]
    c = CacheManager(m.cache_specs(), 16, 8, 4, torch.bfloat16, "cpu")
    assert set(c.groups[0].tensors[c.groups[0].layers[0]]) == {"k4", "ks", "v4", "vs"}


def test_models_that_do_not():
    with pytest.raises(ValueError, match="heads of 64"):
        set_kv_quant(model_of(tiny.TINY["A"][0]), "int4")
    with pytest.raises(ValueError, match="4 bits"):
        set_kv_quant(model_of(ZA), "int4")
    for f in (set_kv_quant, set_weight_quant):
        with pytest.raises(ValueError, match="must be one of"):
            f(model_of(tiny.TINY["D"][0]), "int3")


def test_a_position_encoding_that_writes_the_cache_itself_is_refused():
    from rllm_b200.parts import GQAttention, Part
    with pytest.raises(ValueError, match="does not write"):
        GQAttention(128, 2, 1, 64, Part()).use_kv4()


def test_command_line():
    import argparse
    p = argparse.ArgumentParser()
    cli._model_args(p)
    a = p.parse_args(["--model", "x", "--kv-quant", "int4", "--weight-quant", "int8"])
    cli._refuse_unbuilt(a)
    with pytest.raises(SystemExit, match="not built"):
        cli._refuse_unbuilt(p.parse_args(["--model", "x", "--kv-quant", "int3"]))
    with pytest.raises(SystemExit):
        p.parse_args(["--model", "x", "--weight-quant", "int3"])


def test_no_cpu_path():
    for call in (lambda: quant.quantize_rows(torch.zeros(2, 16)), lambda: quant.quantize_matrix(torch.zeros(2, 16))):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


def test_ranges_of_keys_find_an_sm_each():
    for items in (1, 8, 16, 37, 38, 64, 74, 75, 148, 149, 5000):
        for keys in (1, 300, 600, 1200, 4000, 60000):
            for hd in (64, 128):
                z = quant.portion_parts(items, keys, hd, 148)
                assert z in (1, 2, 4) and (z == 1 or items * z <= 148) and (z == 1 or keys >= 256)
    assert quant.portion_parts(8, 4000, 64, 148) == 4 and quant.portion_parts(64, 2012, 128, 148) == 2


def test_rows_are_checked_when_made():
    codes, scales = torch.zeros(4, 48, dtype=torch.int8), torch.zeros(4)
    assert quant.Int8Rows(codes, scales, 40).shape == (4, 40) and quant.Int8Matrix(codes, scales, 48).dequantize().shape == (4, 48)
    for c, s, width in ((codes, scales, 49), (codes, scales, 32), (codes, scales, 0), (codes.short(), scales, 48), (codes[0], scales, 48),
                        (codes, scales[:3], 48), (codes, scales.double(), 48), (codes[:, :32], scales, 32), (codes, scales[:, None], 48),
                        (codes, torch.zeros(8)[::2], 48)):
        with pytest.raises(ops.KernelError, match="rows in 8 bits"):
            quant.Int8Rows(c, s, width)


def test_the_plain_forms_themselves():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 3, 128, generator=g)
    c, d = Q.groups4(x)
    assert torch.equal(Q.unpack4(Q.pack4(c), d), Q.fake4(x))
    # a group's largest number is held exactly up to its scale's rounding, the others within half a step (7 is the last code)
    far = (Q.fake4(x) - x).abs().unflatten(-1, (-1, 32)) / d.abs()[..., None]
    assert float(far.max()) <= 1.0 + 8 * 2 ** -8 and float(far.median()) < 0.5
    assert float((Q.fake8(x[0]) - x[0]).abs().max()) <= float(x[0].abs().max()) / 254 * (1 + 1e-6)


def test_a_matrix_is_settled_by_its_maker_only():
    """Products read a settled matrix before the kernel in front of them has ended: one put together by a caller, or written to since, is not."""
    m = quant.Int8Matrix(torch.zeros(4, 48, dtype=torch.int8), torch.zeros(4), 48)
    assert not m.settled
    m._settled = m._version()
    assert m.settled
    m.codes[0, 0] = 1
    assert not m.settled
    with torch.inference_mode():
        n = quant.Int8Matrix(torch.zeros(4, 48, dtype=torch.int8), torch.zeros(4), 48)
    assert not n.settled and n._version() == -1
