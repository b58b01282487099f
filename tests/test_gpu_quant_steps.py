"""Whole steps of a model with a cache held in 4 bits, layer by layer: what each layer stores is the plain form's codes of the keys and values that it was
given, and what its attention gives is the plain form's over the numbers that its cache holds, to the kernels' own bounds. A lost key, a wrong
slot or a wrong rounding shows in the layer and step where it happens."""
import pytest
import torch

import plain_llama as P
import plain_quant as Q
import replay
import tiny
from test_gpu_quant import DEV, DT, bound, equal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("family", ["whole", "portions", "mixed", "prefill_then_decode"])
@pytest.mark.parametrize("name", ["D", "E", "F"])
def test_every_layer_of_every_step(name, family, dtype, tmp_path):
    from rllm_b200.engine import load_engine
    d = tiny.make_model_dir(tmp_path, name)
    cfg, _ = P.read_model_dir(d)
    reqs = {f"r{i}": tiny.random_prompt(n, cfg["vocab_size"], 50 + i) for i, n in enumerate((150, 37, 90, 16, 5, 1))}
    steps = getattr(replay, family)(reqs)
    page = tiny.TINY[name][4]
    eng = load_engine(d, dtype=dtype, device=DEV, page_size=page, max_tokens=2 * replay.max_live_tokens(steps, reqs), kv_quant="int4")
    eng.graphs = None                                      # launch by launch, so that every call is seen
    be, dt, seen = eng.backend, DT[dtype], {"stored": 0, "attended": 0}
    attention, store = be.attention, be.kv4_store

    def stored(k, v, cache):
        store(k, v, cache)
        slots = cache.slots.cpu().long()
        live = slots >= 0
        at, off = slots[live] // page, slots[live] % page
        nkv, hd = cache.spec.kv_heads, cache.spec.head_dim
        for n, x in (("k", k), ("v", v)):
            c, s = Q.groups4(x.cpu()[: len(slots)][live].reshape(-1, nkv, hd))
            assert torch.equal(cache.tensors[n + "4"].cpu()[at, :, off], Q.pack4(c)) and equal(cache.tensors[n + "s"].cpu()[at, :, off].double(), s)
        seen["stored"] += int(live.sum())

    def attended(q, cache, ctx, nh, scale, window):
        y = attention(q, cache, ctx, nh, scale, window)
        k, v = (x.cpu().transpose(2, 3).flatten(1, 2).double() for x in be.kv4_read(cache, ctx, torch.float32))
        row, hd = 0, cache.spec.head_dim
        for s, (n, L) in enumerate(zip(ctx.q_lens_host, ctx.kv_lens_host)):
            qs = q[row: row + n].cpu().view(n, nh, hd)
            want, mag, big = Q.attention(qs, k[s, :L], v[s, :L], scale, window)
            got = y[row: row + n].cpu().double().view(n, nh, hd)
            row += n
            assert ((got - want).abs() <= bound(dt, want, mag, big, hd, L, dt == torch.bfloat16 and n > 1)).all()
            seen["attended"] += n
        return y

    be.attention, be.kv4_store = attended, stored
    replay.run_in_process(eng, steps)
    layers = cfg["num_hidden_layers"]
    assert seen == {"stored": layers * sum(map(len, reqs.values())), "attended": layers * sum(map(len, reqs.values()))}
    eng.cache.check()
