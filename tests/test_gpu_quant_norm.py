"""Products in 8 bits with an RMSNorm in front, as every projection and gate/up pair of a quantised model has it, and added into the residual, as every
output and down projection: rows whose quotients lie at whole numbers, so that float's own error moves no code and the bound is float's."""
import pytest
import torch

import plain_quant as Q
from test_gpu_quant import DEV, HALF, ops, quant, rnd

pytestmark = pytest.mark.gpu


def rows_of_codes(R, K, seed):
    """x [R, K] and a norm weight g of powers of two: x g is a code (|c| up to 127, a 127 in every row) times a power of two a row."""
    gen = torch.Generator().manual_seed(seed)
    c = torch.randint(-127, 128, (R, K), generator=gen).double()
    c[:, K // 2] = 127
    g = 2.0 ** torch.randint(-2, 3, (K,), generator=gen).double()
    x = c / g * 2.0 ** torch.randint(-6, 7, (R, 1), generator=gen).double()
    return c, x.float(), g.float()


# streamed from numbers (K up to 4,096), from codes, ranges of K, one CTA a tile, pairs
SIZES = [(1, 300, 64), (3, 2048, 2048), (8, 40, 4096), (7, 500, 1000), (8, 96, 8192), (40, 1000, 4096), (200, 515, 257), (600, 2048, 2048)]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("wdt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,N,K", SIZES)
def test_a_norm_in_front(T, N, K, wdt, gather):
    q, o = quant(), ops()
    c, x, g = rows_of_codes(T + 2, K, T + K)
    rows = torch.randperm(T + 2, generator=torch.Generator().manual_seed(1))[:T] if gather else torch.arange(T)
    w = rnd(2 * N, K, seed=2, dtype=torch.bfloat16)
    m = q.quantize_matrix(w.to(DEV))
    cw, sw = Q.rows8(w)
    n = x.double() * torch.rsqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-5) * g.double()
    s = (n.abs().amax(1) / 127)[rows]
    want = c[rows] @ cw.T * s[:, None] * sw
    args = dict(norm=(g.to(wdt).to(DEV), 1e-5), rows=rows.int().to(DEV) if gather else None)
    xd = (x if gather else x[:T]).to(DEV)
    # the row's scale: a sum of K squares (K / 2 roundings through the root at most), the root (2 of the last place), two products and a division;
    # then the two scales' products
    e = (K / 2 + 8) * 2.0 ** -24
    got = q.linear(xd, m, o.EPI_STORE_F32, **args).cpu().double()
    assert ((got - want).abs() <= e * want.abs()).all()
    got = q.linear(xd, m, o.EPI_STORE, **args).cpu().double()
    assert ((got - want).abs() <= (e + HALF[torch.bfloat16] * 1.01) * want.abs()).all()
    res = rnd(T, 2 * N, seed=9, scale=float(want.abs().mean()))
    got = q.linear(xd, m, o.EPI_ACCUM_F32, res.to(DEV), **args).cpu().double()
    assert ((got - res - want).abs() <= e * want.abs() + 2.0 ** -24 * (res + want).abs() * 1.01).all()
    got = q.linear(xd, m, o.EPI_SWIGLU, out_dtype=torch.float32, **args).cpu().double()
    a, b = want[:, :N], want[:, N:]
    both = a / (1 + torch.exp(-a)) * b
    # silu's slope: a relative error e of a moves silu(a) by e (1 + |a|) of itself at most, the exponential by 2 of its last place
    assert ((got - both).abs() <= (e * (2 + a.abs()) + 8 * 2.0 ** -24) * both.abs() + 1e-30).all()
