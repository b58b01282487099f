"""Attention over a cache held in 4 bits whose values are of very different sizes: places, groups of 32 dimensions, pages, and rows whose weight lies
wholly on small ones. Against the plain 64-bit form, number by number: `bound` is a share of sum_j p_j |v_j| of each dimension, so that a
dimension of small values is held to its own size."""
import math

import pytest
import torch

import plain_quant as Q
from test_gpu_quant import DEV, bound, quant, rnd, run_attention

pytestmark = pytest.mark.gpu

SIZES = ("like", "places", "groups", "pages", "both", "zero_pages", "zero_places", "zero_groups", "small", "large")


def powers(kind, n, nkv, hd, gen):
    """What the values of a sequence are multiplied by, [n, nkv, hd / 32]: powers of two and zeros."""
    one = torch.ones(n, nkv, hd // 32, dtype=torch.float64)
    draw = lambda *shape: 2.0 ** torch.randint(-14, 15, shape, generator=gen).double()
    if kind == "places":
        return one * draw(n, 1, 1)
    if kind == "groups":
        return one * draw(1, nkv, hd // 32)
    if kind == "pages":
        return one * draw(-(-n // 128), 1, 1).repeat_interleave(128, 0)[:n]
    if kind == "both":
        return one * draw(n, 1, 1) * draw(1, nkv, hd // 32)
    if kind == "zero_pages":                                   # and the others small
        return one * 2.0 ** -30 * (torch.arange(n) // 128 % 2).double()[:, None, None]
    if kind == "zero_places":
        return one * (torch.arange(n) % 3 > 0).double()[:, None, None]
    if kind == "zero_groups":
        return one * (torch.randint(0, 3, one.shape, generator=gen) > 0).double()
    return one * {"like": 1.0, "small": 2.0 ** -60, "large": 2.0 ** 60}[kind]


def make(kind, lens, nkv, hd, page=16, seed=0, sink=None):
    """As `make_cache` of the tests beside, values times `powers`. `sink`: every key at these places is the query's own direction."""
    gen = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    t = {n: torch.full((sum(need), nkv, page, hd // 2), 0x5a, dtype=torch.uint8) for n in ("k4", "v4")}
    t.update({n: torch.full((sum(need), nkv, page, hd // 32), math.nan, dtype=torch.bfloat16) for n in ("ks", "vs")})
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    order = torch.randperm(sum(need), generator=gen).tolist()
    held = []
    for s, n in enumerate(lens):
        mine = [order.pop() for _ in range(need[s])]
        table[s, : need[s]] = torch.tensor(mine, dtype=torch.int32)
        at = torch.tensor([mine[j // page] for j in range(n)]), torch.arange(n) % page
        kv = []
        for name in "kv":
            x = torch.randn(n, nkv, hd, generator=gen, dtype=torch.float64)
            if name == "v":
                x = (x.unflatten(-1, (-1, 32)) * powers(kind, n, nkv, hd, gen)[..., None]).flatten(-2)
            elif sink is not None:
                x[[j for j in sink if j < n]] = 3.0
            c, d = Q.groups4(x)
            t[name + "4"][at[0], :, at[1]] = Q.pack4(c)
            t[name + "s"][at[0], :, at[1]] = d.bfloat16()
            kv.append((c.unflatten(-1, (-1, 32)) * d[..., None]).flatten(-2))
        held.append(kv)
    return {n: x.to(DEV) for n, x in t.items()}, table.to(DEV), held


def check(y, q, held, lens, q_lens, nh, hd, scale, window, read_bf16):
    row = 0
    for s, n in enumerate(q_lens):
        want, mag, big = Q.attention(q[row: row + n].cpu().view(n, nh, hd), held[s][0], held[s][1], scale, window)
        got = y[row: row + n].cpu().double().view(n, nh, hd)
        row += n
        tol = bound(torch.bfloat16, want, mag, big, hd, lens[s], read_bf16)
        far = ((got - want).abs() - tol).max()
        assert torch.isfinite(got).all() and far <= 0, (s, float(far), float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("parts", [0, 1, 2, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", SIZES)
def test_portions(kind, hd, parts, monkeypatch):
    """`parts` 0: the kernel of short portions; else that many CTAs share an item's keys. Bound: weights and values rounded to bfloat16, half a
    step each, as `bound` has it for portions; a page in half precision is well within."""
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: max(parts, 1))
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1 if parts else 1 << 30)
    lens, q_lens, nh, nkv = [700, 300], [64, 40], 8, 2
    t, table, held = make(kind, lens, nkv, hd, seed=hd + parts)
    q = rnd(sum(q_lens), nh * hd, seed=6, dtype=torch.bfloat16, scale=1.5).to(DEV)
    for window in (None, 200):
        y, _ = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, hd ** -0.5, window)
        check(y, q, held, lens, q_lens, nh, hd, hd ** -0.5, window, True)


@pytest.mark.parametrize("parts", [0, 2])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["places", "zero_places", "zero_pages", "both"])
def test_portions_whose_weight_lies_on_few_keys(kind, hd, parts, monkeypatch):
    """Queries that a few keys draw nearly all of the weight from: small ones beside large ones, zeros among them."""
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: max(parts, 1))
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1 if parts else 1 << 30)
    lens, q_lens, nh, nkv = [700], [64], 4, 1
    t, table, held = make(kind, lens, nkv, hd, seed=3 * hd + parts, sink=(0, 1, 2, 130, 131, 132, 400))
    q = (0.5 + 0.1 * rnd(64, nh * hd, seed=6)).bfloat16().to(DEV)
    y, _ = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, 16 / hd, None)
    check(y, q, held, lens, q_lens, nh, hd, 16 / hd, None, True)


@pytest.mark.parametrize("parts", [0, 1])
@pytest.mark.parametrize("hd", [64, 128])
def test_portions_of_like_values_keep_half_precision(hd, parts, monkeypatch):
    """Values of one size are half numbers, and so are the weights: with 2^-11 of half a step where bfloat16 has 2^-8. Queries and keys are codes times
    powers of two, so that reading keys as bfloat16 is exact, and few keys share the weight, so that roundings do not average out."""
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: 1)
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1 if parts else 1 << 30)
    L, n, nh, nkv = 600, 128, 4, 1
    t, table, held = make("like", [L], nkv, hd, seed=hd, sink=())
    t["ks"].copy_(torch.where(torch.isnan(t["ks"]), t["ks"], torch.full_like(t["ks"], 0.25)))
    held[0][0] = Q.groups4(held[0][0])[0] * 0.25           # the codes' keys; twelve bits of a value stay
    q = rnd(n, nh * hd, seed=2, scale=1.0).bfloat16().to(DEV)
    y, _ = run_attention(q, t, table, [L], [n], nh, nkv, hd, 16, 4 * hd ** -0.5, None)
    want, mag, big = Q.attention(q.cpu().view(n, nh, hd), held[0][0], held[0][1], 4 * hd ** -0.5, None)
    got = y.cpu().double().view(n, nh, hd)
    # the output's own rounding, half a step of weight and value in half precision (2^-11 each), scores as `bound` has them
    e = torch.expm1(2 * (big * (hd + 6) * 2.0 ** -23 + 1e-5))[..., None] + (L + 16) * 2.0 ** -23 + 2 * 2.0 ** -11
    tol = mag * e * 1.02 + 2.0 ** -8 * want.abs() * 1.02
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (8, 2, 128), (12, 2, 64), (8, 1, 128), (12, 1, 128)])
@pytest.mark.parametrize("kind", SIZES)
def test_single_tokens(kind, nh, nkv, hd):
    """Keys are codes and so exact; the bound has half a step of bfloat16 for a weight, where half precision has 2^-11."""
    lens = [700, 33, 1]
    t, table, held = make(kind, lens, nkv, hd, seed=hd + nh)
    q = rnd(3, nh * hd, seed=6, dtype=torch.bfloat16, scale=1.5).to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for window in (None, 200):
        for splits in (1, 4, 16):
            y = quant().attention_kv4_decode(q, t, lens_d, table, nh, hd ** -0.5, window, 700, splits)
            check(y, q, held, lens, [1, 1, 1], nh, hd, hd ** -0.5, window, False)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["places", "zero_places", "zero_pages", "both"])
def test_single_tokens_whose_weight_lies_on_few_keys(kind, hd):
    lens, nh, nkv = [700], 4, 1
    t, table, held = make(kind, lens, nkv, hd, seed=3 * hd, sink=(0, 1, 2, 130, 131, 132, 400))
    q = (0.5 + 0.1 * rnd(1, nh * hd, seed=6)).bfloat16().to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for splits in (1, 3, 8):
        y = quant().attention_kv4_decode(q, t, lens_d, table, nh, 16 / hd, None, 700, splits)
        check(y, q, held, lens, [1], nh, hd, 16 / hd, None, False)


@pytest.mark.parametrize("kernel", ["short", "long"])
@pytest.mark.parametrize("known", [True, False])
def test_portions_in_a_window_take_scratch_for_what_they_see(known, kernel, monkeypatch):
    """Long contexts of which a window leaves little, at every place of a page of the scratch: numbers of the pages that a row sees any place of."""
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1 if kernel == "long" else 1 << 30)
    lens, q_lens, nh, nkv, hd, window = [9000, 4991, 600, 129], [65, 128, 40, 129], 8, 2, 64, 300
    t, table, held = make("like", lens, nkv, hd, seed=8)
    for s, (L, n) in enumerate(zip(lens, q_lens)):         # as the engine gives pages back
        table[s, : max(0, L - n - window + 1) // 16] = -1
    q = rnd(sum(q_lens), nh * hd, seed=6, dtype=torch.bfloat16, scale=1.5).to(DEV)
    asked = []

    def scratch(size, make):
        asked.append(size)
        return make()
    _, (be, ctx, cache) = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, hd ** -0.5, window)
    if not known:
        ctx.kv_lens_host = None
    ctx.per_forward.clear()
    y = quant().attention_kv4(q, t, ctx, table, nh, hd ** -0.5, window, True, scratch)
    check(y, q, held, lens, q_lens, nh, hd, hd ** -0.5, window, True)
    # 129 + 299 places lie in five pages of 128 at most: k and v of 4 sequences, 2 bytes a number
    assert asked and max(asked) <= 2 * 4 * 5 * nkv * 128 * hd * 2, asked


@pytest.mark.parametrize("entry", [-1, 1 << 20])
@pytest.mark.parametrize("hd,q_lens,dtype", [(64, [1, 1], "bfloat16"), (128, [1, 1], "bfloat16"), (64, [40, 64], "bfloat16"), (128, [64, 1], "bfloat16"),
                                             (64, [1, 40], "float32"), (256, [1, 9], "bfloat16")])
def test_a_visible_place_on_a_page_that_is_not_held_reads_as_zeros(hd, q_lens, dtype, entry, monkeypatch):
    """The engine makes no such call; every form answers it alike: a key and a value of zeros."""
    lens, nh, nkv = [300, 700], 4, 2
    t, table, held = make("like", lens, nkv, hd, seed=5)
    dt = getattr(torch, dtype)
    q = rnd(sum(q_lens), nh * hd, seed=6, dtype=dt, scale=1.5).to(DEV)
    for s, pages in ((0, (3,)), (1, (0, 9, 20, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 31, 32, 33))):
        for p in pages:
            table[s, p] = entry
            for x in held[s]:
                x[16 * p: 16 * p + 16] = 0.0
    for least in (1, 1 << 30):
        monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", least)
        y, _ = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, hd ** -0.5, None)
        row = 0
        for s, n in enumerate(q_lens):
            want, mag, big = Q.attention(q[row: row + n].cpu().view(n, nh, hd), held[s][0], held[s][1], hd ** -0.5)
            got = y[row: row + n].cpu().double().view(n, nh, hd)
            row += n
            tol = bound(dt, want, mag, big, hd, lens[s], dt == torch.bfloat16 and n > 1)
            assert ((got - want).abs() <= tol).all(), (s, float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("window", [None, 150])
@pytest.mark.parametrize("hd,dtype,q_lens", [(64, "bfloat16", [200, 60]), (128, "bfloat16", [200, 60]), (64, "float32", [200, 60]), (64, "bfloat16", [1, 1]),
                                             (128, "bfloat16", [1, 1]), (192, "bfloat16", [60, 1])])
@pytest.mark.parametrize("parts", [0, 1, 2, 4])
def test_values_that_are_not_finite_are_seen_where_they_are_visible_only(hd, dtype, q_lens, window, parts, monkeypatch):
    """A group of a value with a scale of NaN: the group's dimensions are NaN in rows that see the place, and in no other row or dimension."""
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: max(parts, 1))
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1 if parts else 1 << 30)
    lens, nh, nkv = [700, 260], 4, 2
    dt = getattr(torch, dtype)
    t, table, held = make("places", lens, nkv, hd, seed=11)
    gone = [[(3, 0, 1), (540, 1, 0), (600, 0, hd // 32 - 1), (601, 0, 0), (699, 1, 1)], [(100, 1, 1), (259, 0, 0)]]
    for s, places in enumerate(gone):
        for j, head, grp in places:
            t["vs"][int(table[s, j // 16]), head, j % 16, grp] = math.nan
            held[s][1][j, head, 32 * grp: 32 * grp + 32] = 0.0
    q = rnd(sum(q_lens), nh * hd, seed=6, dtype=dt, scale=1.5).to(DEV)
    y, _ = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, hd ** -0.5, window)
    row = 0
    for s, n in enumerate(q_lens):
        want, mag, big = Q.attention(q[row: row + n].cpu().view(n, nh, hd), held[s][0], held[s][1], hd ** -0.5, window)
        got = y[row: row + n].cpu().double().view(n, nh, hd)
        row += n
        nan = torch.zeros(n, nh, hd, dtype=torch.bool)
        for j, head, grp in gone[s]:
            pos = torch.arange(lens[s] - n, lens[s])
            sees = (j <= pos) & (j > pos - window if window else j >= 0)
            nan[:, head * 2: head * 2 + 2, 32 * grp: 32 * grp + 32] |= sees[:, None, None]
        assert torch.equal(torch.isnan(got), nan), s
        tol = bound(dt, want, mag, big, hd, lens[s], dt == torch.bfloat16 and n > 1)
        assert ((got - want).abs() <= tol)[~nan].all(), (s, float(((got - want).abs() / tol)[~nan].max()))


@pytest.mark.parametrize("parts", [0, 1, 2])
@pytest.mark.parametrize("hd", [64, 128])
def test_keys_of_zeros_that_outweigh_small_values(hd, parts, monkeypatch):
    """Nearly all of the weight on keys in pages of zeros, values of 2^-30 elsewhere: what is left of the sum is theirs."""
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: max(parts, 1))
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1 if parts else 1 << 30)
    lens, q_lens, nh, nkv = [700], [64], 4, 1
    t, table, held = make("zero_pages", lens, nkv, hd, seed=7 * hd + parts, sink=(0, 1, 2))
    q = (0.5 + 0.1 * rnd(64, nh * hd, seed=6)).bfloat16().to(DEV)
    y, _ = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, 20 / hd, None)
    check(y, q, held, lens, q_lens, nh, hd, 20 / hd, None, True)


def test_values_of_16_bits_are_refused_without_their_words():
    from rllm_b200.kernels import ops, sm100
    z = lambda *shape, dt=torch.int32: torch.zeros(*shape, dtype=dt, device=DEV)
    k, v, q = z(2, 1, 128, 64, dt=torch.bfloat16), z(2, 1, 128, 64, dt=torch.float16), z(4, 64, dt=torch.bfloat16)
    cu, lens, table = torch.tensor([0, 4], dtype=torch.int32, device=DEV), torch.tensor([100], dtype=torch.int32, device=DEV), z(1, 1)
    vexp, vlost = z(2, 1), z(2, 1, 2, 4)
    fa = lambda v_, **kw: sm100.attention_fa(q, k, v_, cu, lens, table, 4, 4, 100, 1, 0.125, None, **kw)
    tc = lambda v_, **kw: sm100.attention_prefill_tc(q, k, v_, cu, lens, table, 4, 1, 0.125, None, **kw)
    for call in (fa, tc):
        assert not call(v, vexp=vexp, vlost=vlost).any()
        for bad in ({}, {"vexp": vexp}, {"vexp": vexp[:1], "vlost": vlost}, {"vexp": vexp, "vlost": vlost[:1]}, {"vexp": vexp.long(), "vlost": vlost},
                    {"vexp": vexp, "vlost": vlost.cpu()}, {"vexp": vexp, "vlost": vlost.float()}):
            with pytest.raises(ops.KernelError):
                call(v, **bad)
        with pytest.raises(ops.KernelError):
            call(v.bfloat16(), vexp=vexp, vlost=vlost)
