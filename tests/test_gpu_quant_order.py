"""Products in 8 bits whose weight is written just before: by the rows' kernel, which lets the next kernel begin early, with and without a
launch between, and inside a graph. Integer sums are exact, so that the outputs are equal bit for bit."""
import pytest
import torch

from test_gpu_quant import DEV, ops, quant, rnd

pytestmark = pytest.mark.gpu

# (tokens, outputs, numbers): streamed from numbers, streamed from codes, ranges of K, one CTA a tile, pairs of CTAs
SIZES = [(1, 2048, 2048), (8, 16384, 2048), (8, 2048, 8192), (40, 4096, 4096), (256, 16384, 2048), (2048, 8192, 2048)]


@pytest.mark.parametrize("T,N,K", SIZES)
def test_a_weight_written_just_before(T, N, K):
    q, o = quant(), ops()
    ws = [rnd(N, K, seed=i, dtype=torch.bfloat16).to(DEV) for i in range(3)]
    x = rnd(T, K, seed=9, dtype=torch.bfloat16).to(DEV)
    want = []
    for w in ws:
        m = q.quantize_matrix(w)
        assert m.settled
        want.append(q.linear(x, m, o.EPI_STORE_F32))
    xr = q.quantize_rows(x)
    torch.cuda.synchronize()
    codes, scales = torch.empty_like(q.quantize_rows(ws[0]).codes), torch.empty(N, device=DEV)
    got = []
    for i in (0, 1, 2, 1, 0, 2, 2, 0):
        r = q.quantize_rows(ws[i])
        m = q.Int8Matrix(r.codes, r.scales, K)
        assert not m.settled
        got.append((i, q.linear(x, m, o.EPI_STORE_F32)))                # a launch that makes codes may lie between
        r = q.quantize_rows(ws[i])
        got.append((i, q.linear_int8(xr, q.Int8Matrix(r.codes, r.scales, K), o.EPI_STORE_F32)))
        r = q.quantize_rows(ws[i])
        codes.copy_(r.codes)
        scales.copy_(r.scales)
        got.append((i, q.linear_int8(xr, q.Int8Matrix(codes, scales, K), o.EPI_STORE_F32)))
        del r, m
    for i, y in got:
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("T,N,K", [(4, 4096, 2048), (300, 4096, 2048)])
def test_a_weight_quantised_inside_a_graph(T, N, K):
    q = quant()
    w, x = torch.empty(N, K, dtype=torch.bfloat16, device=DEV), rnd(T, K, seed=9, dtype=torch.bfloat16).to(DEV)
    w.copy_(rnd(N, K, seed=1, dtype=torch.bfloat16))
    q.linear(x, q.quantize_matrix(w))                                   # (modules loaded)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m = q.quantize_matrix(w)
        y = q.linear(x, m)
    assert not m.settled
    for i in range(4):
        w.copy_(rnd(N, K, seed=i, dtype=torch.bfloat16))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, q.linear(x, q.quantize_matrix(w)))


def test_a_settled_matrix_that_is_written_again_is_waited_for():
    q = quant()
    w = [q.quantize_matrix(rnd(4096, 2048, seed=i, dtype=torch.bfloat16).to(DEV)) for i in range(2)]
    x = rnd(4, 2048, seed=9, dtype=torch.bfloat16).to(DEV)
    want = q.linear(x, w[1])
    w[0].codes.copy_(w[1].codes)
    w[0].scales.copy_(w[1].scales)
    assert not w[0].settled
    assert torch.equal(q.linear(x, w[0]), want)
    assert w[0].settle().settled and torch.equal(q.linear(x, w[0]), want)
