"""Codewords by their indices and the gradient of that lookup on the GPU (equss_code_lookup, equss_code_lookup_grad) against
plain indexing on the host in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F64, F32 = torch.float64, torch.float32


def indices(num_pq, rows, k, seed, skew=1.0, bad=0.02):
    g = torch.Generator().manual_seed(seed)
    idx = (torch.rand(num_pq, rows, generator=g, dtype=F64) ** skew * k).long().clamp_(max=k - 1)
    out = torch.rand(num_pq, rows, generator=g) < bad
    return torch.where(out, torch.where(torch.rand(num_pq, rows, generator=g) < 0.5, torch.full_like(idx, -1), torch.full_like(idx, k)), idx)


def plain_lookup(idx, books, scale):
    num_pq, k, d = books.shape
    idx = idx.long()
    ok = (idx >= 0) & (idx < k)
    out = torch.stack([books[p][idx[p].clamp(0, k - 1)].to(F32) * scale * ok[p].unsqueeze(1) for p in range(num_pq)], dim=1)
    return out.reshape(idx.shape[1], num_pq * d).to(books.dtype)


def plain_grad(g, idx, k, scale, of=lambda t: t):
    num_pq, rows = idx.shape
    idx = idx.long()
    g3 = of(g.to(F64) * scale).reshape(rows, num_pq, g.shape[1] // num_pq)
    out = torch.zeros(num_pq, k, g3.shape[2], dtype=F64)
    for p in range(num_pq):
        ok = (idx[p] >= 0) & (idx[p] < k)
        out[p].index_add_(0, idx[p][ok], g3[ok, p])
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,num_pq,k,d", [(1, 1, 1, 1), (5, 8, 256, 128), (33, 3, 7, 5), (1000, 16, 64, 16), (129, 1, 3000, 33), (3000, 4, 50, 64),
                                             (77, 2, 9, 768), (65, 1, 12, 4), (500, 3, 20, 127)])
def test_lookup_equals_indexing(rows, num_pq, k, d, dtype, native, dev):
    books = torch.randn(num_pq, k, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    idx = indices(num_pq, rows, k, rows)
    for scale in (1.0, 11.3125, -0.3):
        want = plain_lookup(idx, books, scale)
        for it in (torch.int64, torch.int32, torch.int16):
            got = native.code_lookup(idx.to(it).to(dev), books.to(dev), scale)
            assert got.dtype == dtype and torch.equal(got.cpu(), want), (scale, it)
        by_row = idx.t().contiguous().to(torch.int16).to(dev)             # an index dump's rows
        assert torch.equal(native.code_lookup(by_row.t(), books.to(dev), scale).cpu(), want)
    assert native.code_lookup(idx[:, :0].to(dev), books.to(dev)).shape == (0, num_pq * d)
    one = idx[:, :1].expand(num_pq, 9).to(dev)                              # the same index nine times, stride 0
    assert torch.equal(native.code_lookup(one, books.to(dev)).cpu(), plain_lookup(one.cpu(), books, 1.0))


CASES = [(0, 2, 5, 8), (1, 1, 1, 1), (1, 8, 256, 128), (63, 2, 3, 5), (700, 3, 2500, 16), (2048, 2, 64, 128), (2049, 2, 64, 128), (2300, 5, 1, 32),
         (4100, 1, 2047, 20), (4100, 1, 2048, 20), (5000, 3, 70001, 7), (6000, 2, 40, 300), (9001, 8, 256, 128), (30000, 1, 12, 64), (2500, 1, 5000000, 2),
         (3000, 2, 17, 1), (140000, 1, 300, 8)]


@pytest.mark.parametrize("rows,num_pq,k,d", CASES)
def test_lookup_gradient_is_exact_on_whole_numbers(rows, num_pq, k, d, native, dev):
    """Whole numbers below 2^24 add exactly in any order.  Even, uneven and one-codeword use; codes without rows get zeros."""
    g = torch.randint(-8, 9, (rows, num_pq * d), generator=torch.Generator().manual_seed(rows + d)).to(F32)
    assert rows * 8 * 4 < 2 ** 24
    for skew, bad in ((1.0, 0.02), (4.0, 0.0), (1e9, 0.3), (1.0, 1.0)):
        idx = indices(num_pq, rows, k, 3, skew, bad)
        want = plain_grad(g, idx, k, 4.0).to(F32)
        got = native.code_lookup_grad(g.to(dev), idx.to(dev), k, 4.0)
        assert got.shape == (num_pq, k, d) and torch.equal(got.cpu(), want), (skew, bad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,num_pq,k,d", [(500, 2, 30, 128), (5000, 3, 600, 33), (20000, 4, 256, 64)])
def test_lookup_gradient_within_the_bound_of_its_sum(rows, num_pq, k, d, dtype, native, dev):
    """A product and at most count additions, u each, of a codeword's magnitudes.  Equal calls, index types and layouts give equal
    bits: the order of the sums is fixed by the rows."""
    g = torch.randn(rows, num_pq * d, generator=torch.Generator().manual_seed(1)).to(dtype)
    idx = indices(num_pq, rows, k, 2, 2.0)
    got = native.code_lookup_grad(g.to(dev), idx.to(dev), k, 0.37)
    scale = float(torch.tensor(0.37, dtype=F32))
    count = plain_grad(torch.ones(rows, num_pq), idx, k, 1.0)
    err = (got.cpu().to(F64) - plain_grad(g, idx, k, scale)).abs()
    assert bool((err <= (count + 1) * U * plain_grad(g, idx, k, scale, torch.abs)).all())
    for other in (idx.to(torch.int32), idx.t().contiguous().to(torch.int16).t(), idx):
        assert torch.equal(native.code_lookup_grad(g.to(dev), other.to(dev), k, 0.37), got)
    wide = torch.zeros(rows, num_pq * d + 13, dtype=dtype)
    wide[:, 5:5 + num_pq * d] = g
    assert torch.equal(native.code_lookup_grad(wide.to(dev)[:, 5:5 + num_pq * d], idx.to(dev), k, 0.37), got)
    # a broadcast gradient: every row the same memory
    same = native.code_lookup_grad(g[:1].to(dev).expand(rows, -1), idx.to(dev), k, 1.0)
    assert torch.equal(same, native.code_lookup_grad(g[:1].expand(rows, -1).contiguous().to(dev), idx.to(dev), k, 1.0))


def test_lookup_gradient_keeps_nan_to_its_codeword(native, dev):
    for rows in (300, 5000):
        idx = indices(1, rows, 20, 5, bad=0.1)
        g = torch.randn(rows, 16)
        g[idx[0] == 3] = float("nan")
        g[(idx[0] < 0) | (idx[0] >= 20)] = float("inf")                    # rows of no codeword
        got = native.code_lookup_grad(g.to(dev), idx.to(dev), 20).cpu()
        assert bool(torch.isnan(got[0, 3]).all()) and bool(torch.isfinite(got[0, torch.arange(20) != 3]).all())


def test_lookup_calls_in_replayed_graphs(native, dev):
    """Two graphs of the same calls and eager calls in between: every replay gives the eager result."""
    rows, num_pq, k, d = 4000, 3, 100, 32
    books = torch.randn(num_pq, k, d, device=dev)
    idx = indices(num_pq, rows, k, 7).to(dev)
    g = torch.randn(rows, num_pq * d, device=dev)

    def step():
        return native.code_lookup(idx, books, 2.0), native.code_lookup_grad(g, idx, k, 2.0)

    step()
    graphs, held = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(step())
        graphs.append(graph)
    for i in range(4):
        g.add_(1.0)
        idx.copy_(idx.roll(7, dims=1))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for h in held:
            assert all(torch.equal(x, y) for x, y in zip(h, want)), i
        native.code_lookup_grad(g[:3000], idx[:, :3000], k)
        torch.cuda.synchronize()


@pytest.mark.parametrize("rows,num_pq,k,d", [(70003, 8, 256, 128), (70003, 40, 20, 28), (70003, 4, 2100, 300)])
def test_lookup_gradient_is_exact_where_the_chip_is_full(rows, num_pq, k, d, native, dev):
    """Enough rows for tiles of 64 everywhere, one row in flight a group: rows / 64 of them times sub-spaces times lanes a row, 2^18 or more.
    Whole numbers below 2^24 add exactly in any order."""
    assert (rows + 63) // 64 * num_pq * min(64, (d + 3) // 4) >= 2 ** 18 and rows * 8 * 4 < 2 ** 24
    g = torch.randint(-8, 9, (rows, num_pq * d), generator=torch.Generator().manual_seed(rows + d)).to(F32)
    for skew, bad in ((2.0, 0.02), (1e9, 0.3)):
        idx = indices(num_pq, rows, k, 3, skew, bad)
        want = plain_grad(g, idx, k, 4.0).to(F32)
        got = native.code_lookup_grad(g.to(dev), idx.to(dev), k, 4.0)
        assert torch.equal(got.cpu(), want), skew
