"""Quantised serving on the GPU: rows and products in 8 bits, keys and values held in 4 bits, attention over them, and whole models,
against the plain 64-bit forms. Codes are exact by definition and compared for equality; tolerances of float results are sums of the
roundings on the way (a rounding is off by at most half a step, `torch.finfo(t).eps / 2` of the value)."""
import math

import pytest
import torch

import plain_llama as P
import plain_quant as Q
import replay
import tiny

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def quant():
    from rllm_b200.kernels import quant as q
    return q


def ops():
    from rllm_b200.kernels import ops as o
    return o


def rnd(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def equal(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


# ------------------------------------------------------------------ rows in 8 bits

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (2, 16), (5, 33), (4, 2048), (3, 2056), (2, 4095), (3, 8192), (2, 8193), (2, 14336),
                                 (300, 1111), (1, 40000)])
def test_rows_in_8_bits(T, K, dtype):
    x = rnd(T, K, seed=T + K, dtype=DT[dtype], scale=3.0)
    if T > 2:
        x[1] = 0
        x[2] *= 1e-30
    got = quant().quantize_rows(x.to(DEV))
    c, s = Q.rows8(x)
    assert got.shape == (T, K) and got.codes.shape[1] == -(-K // 16) * 16
    assert torch.equal(got.scales.cpu().double(), s)
    assert torch.equal(got.codes[:, :K].cpu().double(), c) and not got.codes[:, K:].any()


def test_borders_go_to_even():
    """Quotients that are half-integers exactly, and ones a float's last place beside them."""
    half = torch.arange(-126.5, 127.0)
    for s in (1.0, 2.0 ** -120, 3.0, 1.0 / 3, 7.7e20):
        x = (half.double() * torch.tensor(s, dtype=torch.float32).double()).float()
        top = torch.tensor([127.0 * float(torch.tensor(s))], dtype=torch.float32)
        rows = torch.stack([torch.cat([top, f]) for f in (x, torch.nextafter(x, x + x), torch.nextafter(x, torch.zeros_like(x)))])
        got = quant().quantize_rows(rows.to(DEV))
        c, sc = Q.rows8(rows)
        assert torch.equal(got.scales.cpu().double(), sc) and torch.equal(got.codes[:, : rows.shape[1]].cpu().double(), c)


def test_rows_of_every_size_of_number():
    x = torch.stack([rnd(64, seed=i).double() * 2.0 ** e for i, e in enumerate((-140, -130, -100, -30, 0, 60, 120, 125))]).float()
    got = quant().quantize_rows(x.to(DEV))
    c, s = Q.rows8(x)
    assert torch.equal(got.scales.cpu().double(), s)
    # below 2^-126 a quotient of two denormal numbers is still rounded once: at most one code
    assert torch.equal(got.codes[2:, :64].cpu().double(), c[2:]) and float((got.codes[:2, :64].cpu().double() - c[:2]).abs().max()) <= 1


@pytest.mark.parametrize("dtype", list(DT))
def test_rows_that_are_not_finite_become_nan(dtype):
    x = rnd(5, 100, dtype=DT[dtype])
    x[1, 99], x[2, 0], x[3, 50] = math.inf, -math.inf, math.nan
    got = quant().quantize_rows(x.to(DEV))
    assert torch.isnan(got.scales.cpu()).tolist() == [False, True, True, True, False]
    assert torch.isnan(got.dequantize()[1:4]).all() and torch.isfinite(got.dequantize()[[0, 4]]).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("K", [64, 100, 2048, 4097])
def test_rows_with_a_norm_in_front(K, dtype):
    x, g = rnd(9, K, seed=K, scale=4.0), (1 + rnd(K, seed=1, scale=0.3)).to(DT[dtype])
    rows = torch.tensor([8, 0, 3, 3], dtype=torch.int32)
    got = quant().quantize_rows(x.to(DEV), (g.to(DEV), 1e-5), rows.to(DEV))
    n = x.double()[rows.long()]
    n = n * torch.rsqrt((n * n).mean(1, keepdim=True) + 1e-5) * g.double()
    # the float norm is off by its sum (K roundings of positive terms at most, halved by the root), the root (2) and two products
    eps = (K / 2 + 6) * 2.0 ** -24
    s = n.abs().amax(1) / 127
    assert float((got.scales.cpu().double() / s - 1).abs().max()) <= eps + 2.0 ** -23
    far = (got.dequantize().cpu().double() - n).abs() / s[:, None]
    assert float(far.max()) <= 0.5 + 127 * (2 * eps + 2.0 ** -22)


def test_rows_lie_apart():
    x = rnd(6, 200, dtype=torch.bfloat16)
    view = x.to(DEV)[:, 3: 3 + 128]
    got = quant().quantize_rows(view)
    assert torch.equal(got.codes.cpu().double(), Q.rows8(x[:, 3: 131])[0])


# ------------------------------------------------------------------ products in 8 bits

SIZES = [(1, 1, 1), (1, 64, 64), (1, 2048, 2048), (2, 40, 33), (7, 130, 1000), (8, 515, 4096), (9, 256, 512), (16, 96, 8192), (17, 1000, 300),
         (33, 2048, 256), (64, 128, 14336), (65, 72, 96), (128, 513, 640), (129, 384, 1111), (200, 1001, 257), (300, 2050, 512),
         (513, 300, 128), (1000, 260, 2048), (130, 96, 4096), (40, 4096, 4096), (100, 17, 8200), (20, 600, 1024)]


def product_inputs(T, N, K, dtype, seed=0):
    x, w = rnd(T, K, seed=seed + 1, dtype=dtype), rnd(N, K, seed=seed + 2, dtype=torch.bfloat16)
    q = quant()
    return q.quantize_rows(x.to(DEV)), q.quantize_matrix(w.to(DEV)), Q.rows8(x), Q.rows8(w)


def plain_product(x, w):
    (cx, sx), (cw, sw) = x, w
    return (cx @ cw.T) * sx[:, None] * sw


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,N,K", SIZES)
def test_product(T, N, K, dtype):
    dt = DT[dtype]
    x, w, px, pw = product_inputs(T, N, K, dt)
    want = plain_product(px, pw)
    o = ops()
    # the integer sum is exact; it, and its products with two scales, are each rounded to float, then once to the output's type
    e = 3 * 2.0 ** -24 * 1.01
    y = quant().linear_int8(x, w, o.EPI_STORE, out_dtype=dt).cpu().double()
    assert ((y - want).abs() <= (e + HALF[dt]) * want.abs()).all()
    y = quant().linear_int8(x, w, o.EPI_STORE_F32).cpu().double()
    assert ((y - want).abs() <= e * want.abs()).all()
    res = rnd(T, N, seed=5)
    out = res.to(DEV)
    quant().linear_int8(x, w, o.EPI_ACCUM_F32, out)
    total = res.double() + want
    assert ((out.cpu().double() - total).abs() <= e * want.abs() + 2.0 ** -24 * total.abs() * 1.01).all()


# tiles of two SMs: ends of tokens, outputs and K inside a tile, in either of the two, one tile a pair and several
@pytest.mark.parametrize("T,N,K", [(1000, 4601, 4112), (700, 6000, 2500), (2049, 2000, 4100), (1400, 4096, 4112), (300, 9001, 4500),
                                   (4097, 2200, 2060), (1030, 9000, 2000)])
def test_products_of_many_tokens(T, N, K):
    import ctypes
    from rllm_b200.kernels import build
    lib, bn, splits = build.load_library("quant"), ctypes.c_int(), ctypes.c_int()
    x, w, px, pw = product_inputs(T, N, K, torch.bfloat16)
    want, o = plain_product(px, pw), ops()
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    for epi in (o.EPI_STORE, o.EPI_STORE_F32, o.EPI_ACCUM_F32):
        assert lib.rllm_int8_plan(epi, T, N, K, sms, ctypes.byref(bn), ctypes.byref(splits)) == 0 and bn.value == 512
    e = 3 * 2.0 ** -24 * 1.01                       # (as in test_product)
    for dt in DT.values():
        y = quant().linear_int8(x, w, o.EPI_STORE, out_dtype=dt).cpu().double()
        assert ((y - want).abs() <= (e + HALF[dt]) * want.abs()).all()
    res = rnd(T, N, seed=5)
    out = res.to(DEV)
    quant().linear_int8(x, w, o.EPI_ACCUM_F32, out)
    total = res.double() + want
    assert ((out.cpu().double() - total).abs() <= e * want.abs() + 2.0 ** -24 * total.abs() * 1.01).all()
    if N % 2 == 0:
        assert lib.rllm_int8_plan(o.EPI_SWIGLU, T, N // 2, K, sms, ctypes.byref(bn), ctypes.byref(splits)) == 0 and bn.value == 512
        g, u = want.chunk(2, dim=1)
        want = g / (1 + torch.exp(-g)) * u
        e = (3 * (1 + g.abs()) + 3 + 2 * 2 + 2 * 2 + 2) * 2.0 ** -24 * 2             # (as in test_product_swiglu)
        for dt in DT.values():
            y = quant().linear_int8(x, w, o.EPI_SWIGLU, out_dtype=dt).cpu().double()
            assert ((y - want).abs() <= (e + HALF[dt]) * want.abs() + 1e-30).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,N,K", SIZES)
def test_product_swiglu(T, N, K, dtype):
    dt = DT[dtype]
    x, w, px, pw = product_inputs(T, 2 * N, K, dt, seed=7)
    g, u = plain_product(px, pw).chunk(2, dim=1)
    want = g / (1 + torch.exp(-g)) * u
    y = quant().linear_int8(x, w, ops().EPI_SWIGLU, out_dtype=dt).cpu().double()
    # g is off by 3 roundings, which the exponential turns into |g| of them; the exponential itself (2 units), sum, quotient
    # (2 units) and product; a fast quotient and exponential (serving type) 4 units and |g| more of its argument's rounding
    e = (3 * (1 + g.abs()) + 3 + 2 * 2 + 2 * 2 + 2) * 2.0 ** -24 * 2
    assert ((y - want).abs() <= (e + HALF[dt]) * want.abs() + 1e-30).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,N,K", [(1, 1, 8), (1, 48, 2048), (2, 40, 40), (3, 17, 4104), (5, 130, 1000), (8, 515, 8192), (8, 36, 16384), (7, 33, 16392),
                                   (9, 256, 512), (16, 96, 8192), (13, 100, 4096), (16, 72, 2048), (16, 20, 8200), (17, 64, 64), (4, 30, 33),
                                   (1, 4000, 512), (8, 2400, 256)])
def test_product_from_numbers(T, N, K, dtype):
    """The product that quantises its tokens itself (few of them) equals the two calls, every epilogue, with and without a norm."""
    q, o = quant(), ops()
    w = q.quantize_matrix(rnd(2 * N, K, seed=2, dtype=torch.bfloat16).to(DEV))
    x = rnd(T + 3, K, seed=1, dtype=DT[dtype], scale=2.0).to(DEV)
    if T > 3:
        x[1] = 0
        x[2] *= 1e-36
        x[3, 5] = math.inf
    half = q.Int8Matrix(w.codes[:N], w.scales[:N], K)
    g = (1 + rnd(K, seed=5, scale=0.2)).to(DEV)
    rows = torch.arange(T - 1, -1, -1, dtype=torch.int32, device=DEV)
    for kw in ({}, {"rows": rows}):
        a = q.quantize_rows(x if kw else x[:T], **kw)
        for epi, m in ((o.EPI_STORE, half), (o.EPI_STORE_F32, half), (o.EPI_SWIGLU, w)):
            want = q.linear_int8(a, m, epi, out_dtype=DT[dtype])
            got = q.linear(x if kw else x[:T], m, epi, out_dtype=DT[dtype], **kw)
            assert equal(got, want), (epi, kw)
        res = rnd(T, N, seed=9).to(DEV)
        assert equal(q.linear(x if kw else x[:T], half, o.EPI_ACCUM_F32, res.clone(), **kw), q.linear_int8(a, half, o.EPI_ACCUM_F32, res.clone()))
    # a norm in front sums its squares in another order: the row's scale moves by a few units in the last place, a code by a step
    # where it was next to a border
    for gw in (g, g.bfloat16()):
        want = q.linear_int8(q.quantize_rows(x[:T], (gw, 1e-5)), half, o.EPI_STORE_F32).double()
        got = q.linear(x[:T], half, o.EPI_STORE_F32, norm=(gw, 1e-5)).double()
        size = want.abs().nan_to_num().amax(dim=1, keepdim=True)
        assert equal(torch.isnan(got), torch.isnan(want)) and ((got - want).nan_to_num().abs() <= 0.02 * size + 1e-30).all()
        assert float(((got - want).nan_to_num().abs() <= 1e-5 * size).float().mean()) > 0.5


def test_product_into_a_wider_tensor_and_wide_sums():
    x, w, px, pw = product_inputs(20, 48, 96, torch.bfloat16)
    big = torch.full((20, 100), 7.0, dtype=torch.bfloat16, device=DEV)
    quant().linear_int8(x, w, ops().EPI_STORE, big[:, 10:58])
    assert (big[:, :10] == 7).all() and (big[:, 58:] == 7).all()
    assert torch.equal(big[:, 10:58], quant().linear_int8(x, w, ops().EPI_STORE))
    # every product at its largest: 127^2 K is still a whole number below 2^31
    K = 131072
    ones = torch.ones(3, K, dtype=torch.bfloat16, device=DEV)
    far = quant().linear(torch.full((8, 16384), 3.0, device=DEV), quant().quantize_matrix(torch.full((5, 16384), -2.0, device=DEV)), ops().EPI_STORE_F32)
    assert float((far.double() / -(6 * 16384) - 1).abs().max()) <= 6 * 2.0 ** -24
    for T in (3, 40):
        q = quant()
        y = q.linear_int8(q.quantize_rows(ones.expand(3, K).repeat(14, 1)[:T].contiguous()), q.quantize_matrix(-ones), ops().EPI_STORE_F32)
        assert float((y.double() / -K - 1).abs().max()) <= 6 * 2.0 ** -24


@pytest.mark.parametrize("T", [5, 40])
def test_rows_of_nan_stay_in_their_rows(T):
    x, w = rnd(T, 64), rnd(50, 64, seed=1)
    x[1, 5] = math.nan
    w[7, 3] = math.inf
    q = quant()
    for epi in (ops().EPI_STORE, ops().EPI_STORE_F32):
        bad = torch.isnan(q.linear_int8(q.quantize_rows(x.to(DEV)), q.quantize_matrix(w.to(DEV)), epi).cpu())
        assert bad[1].all() and bad[:, 7].all()
        bad[1], bad[:, 7] = False, False
        assert not bad.any()


def test_products_refuse():
    q, o = quant(), ops()
    x, w = q.quantize_rows(rnd(4, 32).to(DEV)), q.quantize_matrix(rnd(6, 32).to(DEV))
    other = q.quantize_matrix(rnd(6, 40).to(DEV))
    for call in (lambda: q.linear_int8(x, other), lambda: q.linear_int8(x.codes, w), lambda: q.linear_int8(x, x),
                 lambda: q.linear_int8(x, w, 9), lambda: q.linear_int8(x, w, o.EPI_ACCUM_F32),
                 lambda: q.linear_int8(x, q.quantize_matrix(rnd(5, 32).to(DEV)), o.EPI_SWIGLU),
                 lambda: q.linear_int8(x, w, o.EPI_STORE, torch.empty(4, 6, device=DEV)),
                 lambda: q.linear_int8(x, w, o.EPI_STORE_F32, torch.empty(3, 6, device=DEV)),
                 lambda: q.linear_int8(x, w, o.EPI_STORE_F32, torch.empty(4, 12, device=DEV)[:, ::2]),
                 lambda: q.linear_int8(q.quantize_rows(torch.zeros(1, 131073, device=DEV)), q.quantize_matrix(torch.zeros(1, 131073, device=DEV))),
                 lambda: q.quantize_rows(torch.zeros(2, 0, device=DEV)), lambda: q.quantize_rows(torch.zeros(4, 4, device=DEV).T[:, ::2]),
                 lambda: q.quantize_rows(torch.zeros(2, 4, device=DEV, dtype=torch.float16)),
                 lambda: q.quantize_rows(torch.zeros(2, 4, device=DEV), (torch.ones(5, device=DEV), 0.1)),
                 lambda: q.quantize_rows(torch.zeros(2, 4, device=DEV), None, torch.zeros(2, device=DEV))):
        with pytest.raises(o.KernelError):
            call()
    assert q.linear_int8(q.quantize_rows(torch.zeros(0, 32, device=DEV)), w).shape == (0, 6)


# ------------------------------------------------------------------ keys and values held in 4 bits

def make_cache(lens, nkv, hd, page, seed=0, extra=2, given_back=None):
    """Sequences of normal numbers stored in scattered pages by the plain form: (tensors, block table, slots of every position,
    keys and values as held, float64). What no sequence owns holds scales of NaN."""
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(need + [1]) + 1), -1, dtype=torch.int32)
    t = {n: torch.full((pages, nkv, page, hd // 2), 0x5a, dtype=torch.uint8) for n in ("k4", "v4")}
    t.update({n: torch.full((pages, nkv, page, hd // 32), math.nan, dtype=torch.bfloat16) for n in ("ks", "vs")})
    held, slots = [], []
    for s, n in enumerate(lens):
        mine = [order.pop() for _ in range(need[s])]
        table[s, : need[s]] = torch.tensor(mine, dtype=torch.int32)
        kv = []
        slot = torch.tensor([mine[j // page] * page + j % page for j in range(n)], dtype=torch.long)
        for i, name in enumerate("kv"):
            x = rnd(n, nkv, hd, seed=seed + 10 * s + i, dtype=torch.bfloat16)
            c, d = Q.groups4(x)
            t[name + "4"][slot // page, :, slot % page] = Q.pack4(c)
            t[name + "s"][slot // page, :, slot % page] = d.bfloat16()
            kv.append((c.unflatten(-1, (-1, 32)) * d[..., None]).flatten(-2))
        held.append(kv)
        slots.append(slot.int())
        if given_back:
            table[s, : given_back[s]] = -1
    return {n: x.to(DEV) for n, x in t.items()}, table.to(DEV), slots, held


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("T,nkv,hd,page", [(1, 1, 64, 16), (5, 3, 128, 7), (17, 8, 64, 16), (64, 2, 192, 32), (33, 1, 256, 5), (700, 4, 128, 16)])
def test_store_and_read(T, nkv, hd, page, dtype):
    q = quant()
    pages = -(-T // page) + 3
    t = {"k4": torch.full((pages, nkv, page, hd // 2), 0x33, dtype=torch.uint8, device=DEV), "v4": None,
         "ks": torch.full((pages, nkv, page, hd // 32), 5.0, dtype=torch.bfloat16, device=DEV), "vs": None}
    t["v4"], t["vs"] = t["k4"].clone(), t["ks"].clone()
    before = {n: x.clone() for n, x in t.items()}
    both = rnd(T, 2 * nkv * hd + 8, seed=T, dtype=DT[dtype])
    both[0] = 0
    if T > 4:
        both[1, 3], both[2, nkv * hd + 40] = math.inf, math.nan
        both[3] = both[3].abs().clamp(max=1.0) * -1
        both[4] *= 1e-38                                     # scales below the smallest normal number
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:T].int()
    skip = T > 1
    if skip:
        slots[T - 1] = -1
    x = both.to(DEV)
    k, v = x[:, : nkv * hd], x[:, nkv * hd: 2 * nkv * hd]
    q.kv4_store(k, v, t, slots.to(DEV))
    live = slots >= 0
    at, off = slots[live].long() // page, slots[live].long() % page
    for name, src in (("k", both[:, : nkv * hd]), ("v", both[:, nkv * hd: 2 * nkv * hd])):
        c, d = Q.groups4(src[live].reshape(-1, nkv, hd))
        assert equal(t[name + "s"].cpu()[at, :, off].double(), d)
        got, want = t[name + "4"].cpu()[at, :, off], Q.pack4(c)
        ok = torch.ones(len(at), dtype=torch.bool)
        if T > 5 and dtype == "float32":
            ok[4] = False                                    # denormal numbers: within a code, below
        assert torch.equal(got[ok], want[ok])
        one = Q.unpack4(got, torch.ones_like(d)) - Q.unpack4(want, torch.ones_like(d))
        assert float(one.abs().max()) <= 1
        rest = torch.ones(pages, page, dtype=torch.bool)
        rest[at, off] = False
        for n in ("4", "s"):                                 # what no slot names stays
            a, b = t[name + n].cpu().transpose(1, 2)[rest], before[name + n].cpu().transpose(1, 2)[rest]
            assert torch.equal(a, b)


@pytest.mark.parametrize("out", list(DT))
@pytest.mark.parametrize("nkv,hd,page", [(1, 64, 16), (3, 128, 5), (2, 256, 32)])
def test_read(nkv, hd, page, out):
    lens = [1, page, 2 * page + 1, 0, 37]
    t, table, _, held = make_cache(lens, nkv, hd, page, given_back=[0, 0, 1, 0, 0])
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    k, v = quant().kv4_read(t, table, lens_d, max(lens), DT[out])
    width = -(-max(lens) // page)
    assert k.shape == (5, width, nkv, page, hd) and k.dtype == DT[out]
    for s, n in enumerate(lens):
        for got, want in zip((k, v), held[s]):
            g = got[s].cpu().transpose(1, 2).reshape(width * page, nkv, hd)
            first = page if s == 2 else 0
            assert torch.equal(g[first: n], want[first:n].to(DT[out])) and not g[n:].any() and not g[:first].any()


def run_attention(q, t, table, lens, q_lens, nh, nkv, hd, page, scale, window):
    """Through the backend, as a mixer calls it."""
    from rllm_b200.engine.context import GroupView, StepContext
    from rllm_b200.kernels.backend import Backend
    from rllm_b200.parts import KV4CacheSpec, LayerCache
    be = Backend(q.dtype, DEV)
    cu = [0]
    for n in q_lens:
        cu.append(cu[-1] + n)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    pos = [L - n + i for L, n in zip(lens, q_lens) for i in range(n)]
    seq = [s for s, n in enumerate(q_lens) for _ in range(n)]
    T = cu[-1]
    ctx = StepContext(backend=be, num_tokens=T, num_seqs=len(lens), token_ids=i32([0] * T), positions=i32(pos), token_seq=i32(seq),
                      cu_q=i32(cu), kv_lens=i32(lens), state_slots=None, q_lens_host=list(q_lens), kv_lens_host=list(lens),
                      state_slots_host=[-1] * len(lens), groups={0: GroupView(i32([-1] * T), table, page)}, max_q_len=max(q_lens),
                      max_kv_len=max(lens))
    cache = LayerCache(KV4CacheSpec(nkv, hd, window), page, None, None, ctx.groups[0].slots, table, True, tensors=t)
    return be.attention(q, cache, ctx, nh, scale, window), (be, ctx, cache)


def bound(dt, out, mag, big, hd, n, read_bf16):
    """How far a float attention may be off: scores by their sum's roundings (hd + 6 of them, of the summed magnitudes) and, where
    keys are read as bfloat16, by half a step of each; a weight by twice its score's error; with tensor cores (bfloat16) each weight
    and each value by half a step; the sums over keys and the last rounding."""
    ds = big * ((hd + 6) * 2.0 ** -23 + (2.0 ** -8 if read_bf16 else 0.0)) + 1e-5
    e = torch.expm1(2 * ds)[..., None] + (n + 16) * 2.0 ** -23
    if dt == torch.bfloat16:
        e = e + 2.0 ** -8 + (2.0 ** -8 if read_bf16 else 0.0)
    return mag * e * 1.02 + HALF[dt] * out.abs() * 1.02 + 1e-30


ATTENTION = [
    # lens, q_lens, nh, nkv, hd, page, window
    ([1], [1], 1, 1, 64, 16, None), ([300], [1], 32, 8, 64, 16, None), ([5, 17, 1, 64, 33, 129], [1] * 6, 8, 2, 64, 16, None),
    ([700, 3, 1025], [1] * 3, 10, 2, 128, 7, None), ([257, 40], [1] * 2, 16, 1, 128, 16, None), ([90, 2000], [1] * 2, 24, 1, 64, 32, None),
    ([500, 20, 333], [1] * 3, 6, 2, 128, 16, 100), ([400, 65], [1] * 2, 4, 4, 64, 8, 1), ([5000], [1], 8, 8, 128, 16, None),
    ([9], [9], 4, 2, 64, 16, None), ([70, 200], [33, 2], 12, 4, 128, 16, None), ([150], [150], 4, 1, 64, 5, 20),
    ([40, 50, 300, 7], [1, 1, 120, 7], 8, 2, 64, 16, None), ([300, 20, 90], [100, 1, 64], 8, 2, 128, 16, 77),
    ([700], [600], 8, 2, 128, 16, None), ([30, 900, 12, 640], [1, 512, 1, 2], 4, 1, 64, 16, 300),
    ([33, 20], [1, 5], 3, 1, 192, 16, None), ([50, 61], [1, 40], 4, 2, 256, 16, 30),
]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("lens,q_lens,nh,nkv,hd,page,window", ATTENTION)
def test_attention(lens, q_lens, nh, nkv, hd, page, window, dtype):
    dt = DT[dtype]
    back = [max(0, (L - n - window + 1) // page) if window else 0 for L, n in zip(lens, q_lens)]
    t, table, _, held = make_cache(lens, nkv, hd, page, seed=len(lens) + hd, given_back=back)
    T = sum(q_lens)
    buf = rnd(T, (nh + 2 * nkv) * hd, seed=4, dtype=dt, scale=1.5).to(DEV)
    scale = hd ** -0.5
    y, _ = run_attention(buf[:, : nh * hd], t, table, lens, q_lens, nh, nkv, hd, page, scale, window)
    assert y.shape == (T, nh * hd) and y.dtype == dt
    row = 0
    for s, n in enumerate(q_lens):
        q = buf[row: row + n, : nh * hd].cpu().view(n, nh, hd)
        want, mag, big = Q.attention(q, held[s][0], held[s][1], scale, window)
        got = y[row: row + n].cpu().double().view(n, nh, hd)
        row += n
        tol = bound(dt, want, mag, big, hd, lens[s], dt == torch.bfloat16 and n > 1)
        assert ((got - want).abs() <= tol).all(), (s, float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,window", [(1, None), (1, 50), (100, None)])
def test_attention_sees_each_key_once(n, window, dtype):
    """One key far ahead of the others decides the output: every position in turn, the newest and the window's oldest among them."""
    nh, nkv, hd, page, L = 4, 2, 64, 16, 300
    t, table, slots, _ = make_cache([L], nkv, hd, page)
    q = torch.ones(n, nh * hd, dtype=DT[dtype], device=DEV)
    rows = torch.zeros(L, nkv * hd, dtype=DT[dtype], device=DEV)
    vals = (torch.arange(L, device=DEV).float()[:, None] % 64 + 1).expand(L, nkv * hd).to(DT[dtype]).contiguous()
    for j in (0, 1, 15, 16, 31, 32, 63, 64, 127, 128, 199, 200, 250, 251, 298, 299):
        k = rows.clone()
        k[j] = 8.0
        quant().kv4_store(k, vals, t, slots[0].to(DEV))
        y, _ = run_attention(q, t, table, [L], [n], nh, nkv, hd, page, 1.0, window)
        last = y[-1].float().cpu()
        seen = window is None or j > L - 1 - window
        want = float(j % 64 + 1) if seen else None
        if seen:
            assert ((last - want).abs() <= 2.0 ** -7 * want).all(), j
        else:
            lo = L - window
            mean = float((torch.arange(lo, L).float() % 64 + 1).mean())
            assert ((last - mean).abs() <= 2.0 ** -6 * mean).all(), j


def test_a_nan_key_is_seen_where_it_is_visible_only():
    nh, nkv, hd, page = 4, 2, 64, 16
    t, table, slots, held = make_cache([100, 90], nkv, hd, page)
    for name in ("ks", "vs"):
        s0 = int(slots[0][20])
        t[name][s0 // page, 1, s0 % page] = math.nan
    q = rnd(2, nh * hd, dtype=torch.bfloat16).to(DEV)
    y, _ = run_attention(q, t, table, [100, 90], [1, 1], nh, nkv, hd, page, 0.125, None)
    assert torch.isnan(y[0, 2 * hd:]).all() and torch.isfinite(y[0, : 2 * hd]).all() and torch.isfinite(y[1]).all()
    y, _ = run_attention(q, t, table, [100, 90], [1, 1], nh, nkv, hd, page, 0.125, 60)
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("window", [None, 333])
@pytest.mark.parametrize("nh,nkv,hd,lens", [(8, 2, 64, [1, 700, 64, 2049]), (12, 1, 128, [1500, 3]), (40, 8, 64, [130]), (4, 4, 128, [900, 0])])
def test_every_number_of_ranges(nh, nkv, hd, lens, window):
    """The ranges that the keys are cut into do not show: any number of them, on any step, and a hint of the lengths that is wrong."""
    t, table, _, held = make_cache(lens, nkv, hd, 16, seed=7)
    S, scale = len(lens), hd ** -0.5
    q = rnd(S, nh * hd, seed=3, dtype=torch.bfloat16, scale=1.5).to(DEV)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    room = torch.full((S, nh * hd + 24), 7.0, dtype=torch.bfloat16, device=DEV)
    for splits in (None, 1, 2, 3, 4, 5, 6, 7, 8, 16):
        for hint in ((1, 100000) if splits is None else (max(lens),)):
            room.fill_(7.0)
            quant().attention_kv4_decode(q, t, lens_d, table, nh, scale, window, hint, splits, out=room[:, : nh * hd])
            assert (room[:, nh * hd:] == 7.0).all()
            for s, n in enumerate(lens):
                got = room[s, : nh * hd].cpu().double().view(1, nh, hd)
                if n == 0:
                    assert not got.any()
                    continue
                want, mag, big = Q.attention(q[s].cpu().view(1, nh, hd), held[s][0], held[s][1], scale, window)
                tol = bound(torch.bfloat16, want, mag, big, hd, n, False)
                assert ((got - want).abs() <= tol).all(), (splits, hint, s, float(((got - want).abs() / tol).max()))
    for splits in (0, -1, 9, 15, 17):
        with pytest.raises(ops().KernelError):
            quant().attention_kv4_decode(q, t, lens_d, table, nh, scale, window, max(lens), splits)


def test_portions_one_by_one_and_without_scratch(monkeypatch):
    """Portions whose numbers do not fit the scratch at once go one by one; where there is no room for one they are attended over in 4 bits."""
    lens, q_lens, nh, nkv, hd = [700, 20, 640, 577], [100, 1, 200, 64], 8, 2, 64
    t, table, _, _ = make_cache(lens, nkv, hd, 16)
    q = rnd(sum(q_lens), nh * hd, seed=2, dtype=torch.bfloat16).to(DEV)
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: 2)        # (how many ranges of keys there are goes with the run's items)
    call = lambda: run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, 0.125, None)
    y, (be, ctx, cache) = call()
    monkeypatch.setattr(quant(), "READ_BYTES", 1)
    assert torch.equal(call()[0], y)                       # (the same kernels over the same numbers)
    ctx.per_forward.clear()
    ctx.kv_lens_host = None
    assert torch.equal(be.attention(q, cache, ctx, nh, 0.125, None), y)
    simt = quant().attention_kv4(q, t, ctx, table, nh, 0.125, None, True, lambda size, make: None)
    assert torch.equal(simt, quant().attention_kv4_simt(q, t, ctx.token_seq, ctx.positions, table, nh, 0.125))


@pytest.mark.parametrize("parts", [1, 2, 4])
@pytest.mark.parametrize("lens,q_lens,nh,nkv,hd,window", [
    ([700], [64], 8, 2, 64, None), ([520], [32], 8, 2, 128, None), ([1500, 513], [200, 130], 8, 2, 64, None), ([2000], [300], 4, 1, 128, 700),
    ([600], [600], 8, 2, 64, None), ([900], [257], 8, 2, 128, None), ([1030, 520], [33, 520], 16, 2, 64, 100)])
def test_portions_share_their_keys(lens, q_lens, nh, nkv, hd, window, parts, monkeypatch):
    """Ranges of a work item's keys in CTAs of their own: every number of them, ranges that a row tile sees nothing of, rows in short of a tile."""
    monkeypatch.setattr(quant(), "portion_parts", lambda *a: parts)
    monkeypatch.setattr(quant().sm100, "TC_ATTENTION_MIN_KEYS", 1)
    back = [max(0, (L - n - window + 1) // 16) if window else 0 for L, n in zip(lens, q_lens)]
    t, table, _, held = make_cache(lens, nkv, hd, 16, seed=9, given_back=back)
    q = rnd(sum(q_lens), nh * hd, seed=6, dtype=torch.bfloat16, scale=1.5).to(DEV)
    scale, row = hd ** -0.5, 0
    y, _ = run_attention(q, t, table, lens, q_lens, nh, nkv, hd, 16, scale, window)
    for s, n in enumerate(q_lens):
        want, mag, big = Q.attention(q[row: row + n].cpu().view(n, nh, hd), held[s][0], held[s][1], scale, window)
        got = y[row: row + n].cpu().double().view(n, nh, hd)
        row += n
        tol = bound(torch.bfloat16, want, mag, big, hd, lens[s], True)
        assert ((got - want).abs() <= tol).all(), (s, float(((got - want).abs() / tol).max()))


def test_calls_of_nothing():
    q, o = quant(), ops()
    none = torch.zeros(0, 128, device=DEV, dtype=torch.bfloat16)
    w = q.quantize_matrix(rnd(40, 128, dtype=torch.bfloat16).to(DEV))
    assert q.quantize_rows(none).shape == (0, 128) and q.linear(none, w).shape == (0, 40) and q.linear(none, w, o.EPI_SWIGLU).shape == (0, 20)
    assert q.linear_int8(q.quantize_rows(none), w, o.EPI_STORE_F32).shape == (0, 40)
    x = rnd(3, 128, dtype=torch.bfloat16).to(DEV)
    assert q.linear(x, w, rows=torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 40)
    t, table, _, _ = make_cache([20], 2, 64, 16)
    i32 = torch.zeros(0, dtype=torch.int32, device=DEV)
    before = {n: a.clone() for n, a in t.items()}
    q.kv4_store(none, none, t, i32)
    assert all(torch.equal(a.view(torch.uint8), before[n].view(torch.uint8)) for n, a in t.items())
    assert q.attention_kv4_simt(none, t, i32, i32, table, 2, 1.0).shape == (0, 128)
    assert q.attention_kv4_decode(none, t, i32, table, 2, 1.0, None, 1).shape == (0, 128)
    torch.cuda.synchronize()


@pytest.mark.parametrize("T", [1, 8, 40, 700])
def test_captured_and_replayed(T):
    """A layer's calls, captured together on a stream of their own, replayed over new inputs: the same numbers as launch by launch. Two graphs
    replayed at once on two streams do not disturb one another."""
    q, o, nh, nkv, hd = quant(), ops(), 8, 2, 64
    lens = [64 + 5 * (i % 40) for i in range(min(T, 40))]
    t, table, slots, _ = make_cache(lens, nkv, hd, 16)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=DEV)
    last = torch.tensor([int(s[-1]) for s in slots], dtype=torch.int32, device=DEV)
    w = [q.quantize_matrix(rnd(n, k, seed=n, dtype=torch.bfloat16).to(DEV)) for n, k in ((12 * 64, 512), (512, 512), (2 * 1024, 512), (512, 1024))]
    S = len(lens)

    def layer(x, cache):
        qkv = q.linear(x, w[0])
        q.kv4_store(qkv[:S, 512: 640], qkv[:S, 640:], cache, last)
        a = q.attention_kv4_decode(qkv[:S, :512], cache, lens_d, table, nh, 0.125, None, 300)
        h = q.linear(torch.cat([a, x[S:]]), w[1], o.EPI_STORE_F32)
        f = q.linear(x, w[2], o.EPI_SWIGLU)
        q.linear(f, w[3], o.EPI_ACCUM_F32, h)
        return h

    caches = [{n: a.clone() for n, a in t.items()} for _ in range(2)]
    xs = [rnd(T, 512, seed=i, dtype=torch.bfloat16).to(DEV) for i in range(4)]
    want = [layer(x, {n: a.clone() for n, a in t.items()}).clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    ins = [torch.zeros_like(xs[0]) for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(layer(ins[i], caches[i]))
        graphs.append(g)
    for a, b in ((0, 1), (2, 3), (1, 0)):
        for i, n in enumerate((a, b)):
            ins[i].copy_(xs[n])
        torch.cuda.synchronize()
        for _ in range(5):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[b])


def test_cache_calls_refuse():
    q, o = quant(), ops()
    t, table, slots, _ = make_cache([20], 2, 64, 16)
    x, sl = torch.zeros(20, 128, device=DEV, dtype=torch.bfloat16), slots[0].to(DEV)
    lens = torch.tensor([20], dtype=torch.int32, device=DEV)
    i32 = torch.zeros(1, dtype=torch.int32, device=DEV)
    narrow = {n: a[..., : a.shape[-1] // 2].contiguous() for n, a in t.items()}
    for call in (lambda: q.kv4_store(x[:, :64], x[:, :64], t, sl), lambda: q.kv4_store(x, x[:5], t, sl), lambda: q.kv4_store(x, x.float(), t, sl),
                 lambda: q.kv4_store(x, x, t, sl.long()), lambda: q.kv4_store(x, x, t, sl[:5]), lambda: q.kv4_store(x, x, narrow, sl),
                 lambda: q.kv4_store(x, x, dict(t, ks=t["ks"].float()), sl), lambda: q.kv4_store(x, x, dict(t, v4=t["v4"][:1]), sl),
                 lambda: q.kv4_store(x.half(), x.half(), t, sl),
                 lambda: q.kv4_read(t, table, lens, 100), lambda: q.kv4_read(t, table.long(), lens, 20),
                 lambda: q.attention_kv4_simt(torch.zeros(1, 3 * 64, device=DEV), t, i32, i32, table, 3, 1.0),
                 lambda: q.attention_kv4_simt(torch.zeros(1, 100, device=DEV), t, i32, i32, table, 2, 1.0),
                 lambda: q.attention_kv4_decode(x[:1], t, lens, table, 2, 0.0, None, 20),
                 lambda: q.attention_kv4_decode(x[:1].float(), t, lens, table, 2, 1.0, None, 20),
                 lambda: q.attention_kv4_decode(x[:1], t, lens, table, 2, 1.0, None, 20, out=x[:1].float()),
                 lambda: q.attention_kv4_decode(x[:1], t, lens, table, 2, 1.0, None, 20, out=x[:2]),
                 lambda: q.attention_kv4_decode(x[:1], t, lens, table, 2, 1.0, None, 20, out=x[:1].cpu())):
        with pytest.raises(o.KernelError):
            call()


# ------------------------------------------------------------------ together: whole models

@pytest.fixture(scope="module")
def dirs(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    return {n: tiny.make_model_dir(root, n) for n in "DEF"}


def traces(name, dirs):
    cfg, w = P.read_model_dir(dirs[name])
    reqs = {f"r{i}": tiny.random_prompt(n, cfg["vocab_size"], 50 + i) for i, n in enumerate((150, 37, 90, 16, 5, 1))}
    return cfg, w, reqs


def rows(got, rid, toks):
    return torch.stack([torch.as_tensor(got[(rid, i)]) for i in range(len(toks))]).double()


CHOICES = [("D", "int4", "none"), ("D", "none", "int8"), ("D", "int4", "int8"), ("E", "int4", "int8"), ("F", "int4", "int8")]


@pytest.mark.parametrize("name,kv,wq", CHOICES)
def test_models_in_32_bits(name, kv, wq, dirs):
    """Against the plain 64-bit form, request by request. A number next to a border between two codes falls on its other side in
    float with a probability of about 2e-5 a code (a float norm is off by some 3e-7, a code of 30 then by 1e-5 on either side), and
    with some 2,200 codes a token that happens to one token in twenty: of 24 requests of four tokens about four in five are untouched and
    agree to float's own error (2e-5); one that is not has a step of a code somewhere, and stays as near as the quantised model is to
    the model itself. E's norm weights are all 1, so that its first layer's quotients are 127 x / m with x and m bfloat16: x = m / 2 is
    the half-integer 63.5 exactly, and a float norm leaves it on either side. A number of 136 is such a one, of either sign, with a
    probability of about 2^-8 / 2 (one cell of 2^-8 of its size, at half the maximum, a density of one third there): one token in four,
    and a third of the requests (0.75^4) have none; a plain form in 32-bit torch finds the same 8 of 24."""
    from rllm_b200.engine import load_engine
    cfg, w = P.read_model_dir(dirs[name])
    reqs = {f"r{i}": tiny.random_prompt(4, cfg["vocab_size"], 50 + i) for i in range(24)}
    eng = load_engine(dirs[name], dtype="float32", device=DEV, page_size=tiny.TINY[name][4], max_tokens=512, kv_quant=kv, weight_quant=wq)
    got = replay.run_in_process(eng, replay.mixed(reqs, decode_tail=2))
    far = []
    for rid, toks in reqs.items():
        want, plain = Q.llama(cfg, w, toks, kv4=kv == "int4", int8=wq == "int8"), Q.llama(cfg, w, toks)
        far.append(float((rows(got, rid, toks) - want).abs().max() / want.abs().max()))
        assert far[-1] <= float((want - plain).abs().max() / want.abs().max()), rid
    assert sum(f <= 2e-5 for f in far) >= (4 if name == "E" else 12), sorted(far)
    eng.cache.check()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("family", ["whole", "portions", "mixed", "prefill_then_decode"])
@pytest.mark.parametrize("name,kv,wq", CHOICES)
def test_models_in_every_way_of_cutting(name, kv, wq, family, dtype, dirs):
    """Long requests, where a moved code moves what later tokens quantise: two runs of the quantised model whose codes differ in places
    are never further apart than quantised and plain model are, which is the sum of all codes' errors."""
    from rllm_b200.engine import load_engine
    cfg, w, reqs = traces(name, dirs)
    steps = getattr(replay, family)(reqs)
    eng = load_engine(dirs[name], dtype=dtype, device=DEV, page_size=tiny.TINY[name][4],
                      max_tokens=2 * replay.max_live_tokens(steps, reqs), kv_quant=kv, weight_quant=wq)
    got = replay.run_in_process(eng, steps)
    far = own = 0.0
    for rid, toks in reqs.items():
        want = Q.llama(cfg, w, toks, kv4=kv == "int4", int8=wq == "int8")
        far += float((rows(got, rid, toks) - want).square().sum())
        own += float((want - Q.llama(cfg, w, toks)).square().sum())
    assert math.sqrt(far / own) <= 1.0, math.sqrt(far / own)
    eng.cache.check()


def test_generate_and_graphs(dirs):
    """`LLM(kv_quant=, weight_quant=)`: steps in graphs and launch by launch draw the same tokens, alone or side by side."""
    from rllm_b200.api import LLM
    from rllm_b200.sampling import SamplingParams
    cfg, _ = P.read_model_dir(dirs["D"])
    prompts = [tiny.random_prompt(n, cfg["vocab_size"], n) for n in (40, 3, 77)]
    sp = SamplingParams(temperature=0.0, max_tokens=24, ignore_eos=True)
    outs = []
    for graphs in (True, False):
        llm = LLM(dirs["D"], num_pages=64, kv_quant="int4", weight_quant="int8")
        if not graphs:
            llm.engine.graphs = None
        outs.append(llm.generate(prompts, sp))
        assert (llm.engine.graph_steps > 0) == graphs
        llm.engine.check()
        llm.engine.cache.check()
    assert outs[0] == outs[1]


def test_the_command_line_runs_it(dirs, capsys):
    from rllm_b200 import cli
    args = ["run", "--model", str(dirs["D"]), "--prompt-ids", "3,7,11,2", "--max-tokens", "5", "--temperature", "0"]
    for more in ([], ["--kv-quant", "int4"], ["--weight-quant", "int8"], ["--kv-quant", "int4", "--weight-quant", "int8"]):
        assert not cli.main(args + more)
        assert capsys.readouterr().out.strip()


def test_a_second_engine_of_the_same_model(dirs):
    from rllm_b200.engine import Entry, load_engine
    from rllm_b200.engine.factory import make_engine
    a = load_engine(dirs["D"], device=DEV, num_pages=16, kv_quant="int4", weight_quant="int8")
    b = make_engine(a.model, num_pages=16, dtype="bfloat16", device=DEV, kv_quant="int4", weight_quant="int8")
    toks = tiny.random_prompt(40, P.read_model_dir(dirs["D"])[0]["vocab_size"], 3)
    x, y = (e.step([Entry("a", toks, [39])]).clone() for e in (a, b))
    assert torch.equal(x, y)


def test_the_cache_takes_less(dirs):
    from rllm_b200.engine import load_engine
    a, b = (load_engine(dirs["D"], device=DEV, num_pages=8, kv_quant=k) for k in ("none", "int4"))
    size = lambda e: sum(t.nbytes for g in e.cache.groups for ts in g.tensors.values() for t in ts.values())
    assert size(b) * 32 == size(a) * 9


def test_per_operation_timing_knows_quantised_models(dirs, monkeypatch, capsys):
    monkeypatch.setenv("RLLM_B200_PROFILE", "1")
    from rllm_b200.engine import Entry, load_engine
    eng = load_engine(dirs["D"], device=DEV, num_pages=16, kv_quant="int4", weight_quant="int8")
    eng.step([Entry("a", [1, 2, 3], [2])])
    eng.step([Entry("a", [4], [0])])
    r = eng.backend.report()
    assert {"qkv+rope", "attention", "gate_up", "down"} <= set(r) and all(c["gbs"] > 0 for n, c in r.items() if n != "norm")
