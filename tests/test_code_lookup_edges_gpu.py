"""The codeword lookup and its gradient at the sizes and uses that their variants part at, and forward-mode differentiation."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

pytestmark = pytest.mark.gpu

F64 = torch.float64
U = 2.0 ** -24


def test_lookup_carries_tangents(pkg, dev):
    """The lookup is linear in the books: its tangent is the lookup of the tangent, and its gradient's tangent the gradient of
    the tangent."""
    torch.manual_seed(21)
    books, t = torch.randn(3, 20, 24, device=dev), torch.randn(3, 20, 24, device=dev)
    idx = torch.randint(-1, 21, (3, 500), device=dev)
    with fwd.dual_level():
        out, tangent = fwd.unpack_dual(pkg.code_lookup(idx, fwd.make_dual(books, t), 1.5))
        assert torch.equal(out, pkg.code_lookup(idx, books, 1.5)) and torch.equal(tangent, pkg.code_lookup(idx, t, 1.5))
    # forward over reverse: d/ds of the gradient of <lookup(B)^2, 1> at B + s t is 2 lookup^T lookup t
    with fwd.dual_level():
        dual = fwd.make_dual(books.clone().requires_grad_(True), t)
        (grad,) = torch.autograd.grad(pkg.code_lookup(idx, dual, 1.0).square().sum(), dual, create_graph=True)
        tangent = fwd.unpack_dual(grad).tangent
    counts = torch.stack([torch.bincount(r[(r >= 0) & (r < 20)], minlength=20) for r in idx]).float().unsqueeze(-1)
    # (a product with a whole number by repeated addition: at most count additions of u each)
    assert bool(((tangent - 2 * counts * t).abs() <= (counts + 2) * U * (2 * counts * t).abs()).all())


@pytest.mark.parametrize("normalize", ["z_norm", "none"])
def test_training_quantiser_carries_tangents(normalize, pkg, dev):
    """The quantiser's z_norm / none training branch with a dual codebook: the vq loss's tangent is its directional difference."""
    torch.manual_seed(22)
    p, k, d, n = 1, 32, 32, 200
    rows = torch.randn(n, d, device=dev)
    books, t = torch.randn(p, k, d, device=dev), torch.randn(p, k, d, device=dev)

    def loss(b):
        return pkg.pqgo._quantize_rows(rows, b, normalize, 0.25, 1.0, True, None)[2]["vq-loss"]

    with fwd.dual_level():
        tangent = fwd.unpack_dual(loss(fwd.make_dual(books.clone().requires_grad_(True), t))).tangent
    b = books.clone().requires_grad_(True)
    (grad,) = torch.autograd.grad(loss(b), b)
    # both are sums of n d products in fp32, in different orders: n d u of the magnitudes' sum at most
    assert abs(float((grad.to(F64) * t.to(F64)).sum() - tangent.detach().to(F64))) <= n * d * U * float((grad.abs().to(F64) * t.abs().to(F64)).sum())


def test_vector_quantizer_carries_tangents(pkg, dev):
    torch.manual_seed(23)
    vq = pkg.quantizer.VectorQuantizer(num_codebook=32, embed_dim=32, normalize="none").to(dev).train()
    z, t = torch.randn(2, 32, 5, 5, device=dev), torch.randn(32, 32, device=dev)
    (grad,) = torch.autograd.grad(vq(z)[1]["loss"], vq.codebook.weight)
    weight = vq.codebook.weight.detach().clone()
    del vq.codebook.weight
    with fwd.dual_level():
        vq.codebook.weight = fwd.make_dual(weight.requires_grad_(True), t)
        tangent = fwd.unpack_dual(vq(z)[1]["loss"]).tangent
    assert abs(float((grad.to(F64) * t.to(F64)).sum() - tangent.detach().to(F64))) <= 1600 * U * float((grad.abs().to(F64) * t.abs().to(F64)).sum())


def clustered(kind, num_pq, rows, k, seed):
    g = torch.Generator().manual_seed(seed)
    near = torch.randint(0, k, (num_pq, rows), generator=g)
    if kind == "low":                                       # a vocabulary in the order of its frequency
        near = (torch.rand(num_pq, rows, generator=g, dtype=F64) ** 6 * k).long().clamp_(max=k - 1)
    elif kind == "cluster":
        near = torch.randint(0, min(k, 300), (num_pq, rows), generator=g)
    elif kind == "busy":                                    # a tenth of the rows on the last code, a tenth on its neighbour
        u = torch.rand(num_pq, rows, generator=g)
        near = torch.where(u < 0.1, torch.full_like(near, k - 1), torch.where(u < 0.2, torch.full_like(near, max(k - 2, 0)), near))
    elif kind == "padding":
        near = torch.where(torch.rand(num_pq, rows, generator=g) < 0.4, torch.full_like(near, -1), near)
    elif kind == "pairs":                                   # runs on either side of the border between one group's and all groups'
        near = (torch.arange(rows) // 64 + torch.arange(rows) // 129).clamp_(max=k - 1).repeat(num_pq, 1)
    return near


@pytest.mark.parametrize("rows,num_pq,k,d", [(257, 1, 5000, 4), (2048, 1, 40000, 3), (2048, 2, 2000, 8), (4096, 1, 150000, 32), (4095, 2, 16384, 16),
                                             (4096, 1, 2000000, 2), (3000, 1, 70000, 128), (2000, 1, 3000, 700), (1999, 3, 900, 60), (600, 1, 1, 24)])
def test_lookup_gradient_of_few_rows_on_neighbouring_codes(rows, num_pq, k, d, native, dev):
    """More than 256 rows on the codes of one workgroup, in every mixture of long and short runs.  Whole numbers add exactly."""
    g = torch.randint(-8, 9, (rows, num_pq * d), generator=torch.Generator().manual_seed(rows)).float()
    for kind in ("low", "cluster", "busy", "padding", "pairs"):
        idx = clustered(kind, num_pq, rows, k, 31)
        want = torch.zeros(num_pq, k, d)
        for p in range(num_pq):
            ok = idx[p] >= 0
            want[p].index_add_(0, idx[p][ok], g.reshape(rows, num_pq, d)[ok, p])
        got = native.code_lookup_grad(g.to(dev), idx.to(dev), k)
        assert torch.equal(got.cpu(), want), kind
        x = torch.randn(rows, num_pq * d, device=dev)
        assert torch.equal(native.code_lookup_grad(x, idx.to(dev), k), native.code_lookup_grad(x, idx.to(dev), k)), kind


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,num_pq,k,d", [(4096, 1, 5000, 16), (2048, 2, 2000, 32), (1500, 1, 1800, 128), (1000, 4, 700, 64)])
def test_quantiser_backward_of_few_rows_on_neighbouring_codes(rows, num_pq, k, d, fmt, native, dev):
    """The same for the quantiser's backward, whose rows have gradients of their own, those of no codeword among them: each row's
    is what the call gives for these rows without the clustering (its own to the bit), the codebooks' agree with fp64 sums."""
    for kind in ("low", "cluster", "busy", "padding", "pairs"):
        idx = clustered(kind, num_pq, rows, k, 32)
        g = torch.Generator().manual_seed(33)
        z, g_zq = torch.randn(rows, num_pq * d, generator=g), torch.randn(rows, num_pq * d, generator=g) * 1e-3
        books = torch.randn(num_pq, k, d, generator=g) * d ** -0.5
        kept, gv = native.ckpt_pack(z.to(dev), fmt), torch.tensor(0.7, device=dev)
        gz, gb = native.pq_st_backward_ckpt(kept, books.to(dev), idx.to(dev), g_zq.to(dev), gv, 0.25, 1.5)
        # rows one by one through codebooks of their own: codeword r is row r's
        own = torch.stack([torch.where((idx[p] >= 0).unsqueeze(1), books[p][idx[p].clamp(min=0)], torch.zeros(1, d)) for p in range(num_pq)])
        each = torch.arange(rows).repeat(num_pq, 1)
        apart, _ = native.pq_st_backward_ckpt(kept, own.to(dev), each.to(dev), g_zq.to(dev), gv, 0.25, 1.5)
        assert torch.equal(gz, apart), kind
        z3 = native.ckpt_unpack(kept).cpu().to(F64).reshape(rows, num_pq, d)
        zn, s = z3 / z3.norm(dim=-1, keepdim=True), 0.7 * 2.0 / (rows * num_pq * d) * 1.5
        for p in range(num_pq):
            ok, i = idx[p] >= 0, idx[p].clamp(min=0)
            want, size, count = torch.zeros(k, d, dtype=F64), torch.zeros(k, d, dtype=F64), torch.bincount(i[ok], minlength=k).to(F64).unsqueeze(1)
            want.index_add_(0, i[ok], s * (books[p][i[ok]].to(F64) - zn[ok, p]))
            size.index_add_(0, i[ok], s * (books[p][i[ok]].to(F64).abs() + zn[ok, p].abs()))
            assert bool(((gb[p].cpu().to(F64) - want).abs() <= (count + 16) * U * size).all()), kind   # 16 u a term, u an addition


def test_lookup_gradient_of_more_codes_than_one_launch_joins(native, dev):
    """67 million codes and a few more: the codes behind the first launch's are written like the others, zeros included."""
    rows, k, d = 4200, (1 << 26) + 5, 2
    g = torch.randint(-8, 9, (rows, d), generator=torch.Generator().manual_seed(41)).float()
    last = torch.tensor([0, 1, (1 << 26) - 5, (1 << 26) - 4, (1 << 26) - 3, 1 << 26, k - 2, k - 1, k, -1])
    idx = last[torch.randint(0, len(last), (1, rows), generator=torch.Generator().manual_seed(42))]
    got = native.code_lookup_grad(g.to(dev), idx.to(dev), k)
    ok = (idx[0] >= 0) & (idx[0] < k)
    want = torch.zeros(1, k, d, device=dev)
    want[0].index_add_(0, idx[0][ok].to(dev), g[ok].to(dev))          # whole numbers: exact in any order
    assert torch.equal(got, want) and int((got != 0).any(-1).sum()) >= 7


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("num_pq,d", [(1, 1 << 18), (1, 1 << 20), (2, 1 << 19)])
def test_lookup_of_the_widest_codewords(num_pq, d, dtype, native, dev):
    """Codewords whose 16-byte units pass the range of the division by multiplication."""
    books = torch.randn(num_pq, 3, d, generator=torch.Generator().manual_seed(43)).to(dtype)
    idx = torch.tensor([[2, 0, -1, 1, 3]]).repeat(num_pq, 1)
    got = native.code_lookup(idx.to(dev), books.to(dev), 0.5).cpu().reshape(5, num_pq, d)
    for r, k in enumerate(idx[0].tolist()):
        want = (books[:, k].float() * 0.5).to(dtype) if 0 <= k < 3 else torch.zeros(num_pq, d, dtype=dtype)
        assert torch.equal(got[r], want), r
    g = torch.ones(5, num_pq * d, dtype=dtype, device=dev)
    assert torch.equal(native.code_lookup_grad(g, idx.to(dev), 3).cpu(), torch.ones(num_pq, 3, d))


@pytest.mark.parametrize("rows,num_pq,k,d", [(3000, 1, 300, 2000), (2500, 1, 1000, 1100), (5000, 2, 40, 1500), (9000, 1, 2100, 515)])
def test_lookup_gradient_of_wide_codewords_is_exact_on_whole_numbers(rows, num_pq, k, d, native, dev):
    """Rows of several waves, on either side of the border between the joins of 16 and of four waves a code."""
    g = torch.randint(-8, 9, (rows, num_pq * d), generator=torch.Generator().manual_seed(44)).float()
    for kind in ("low", "busy", "padding"):
        idx = clustered(kind, num_pq, rows, k, 45)
        want = torch.zeros(num_pq, k, d)
        for p in range(num_pq):
            ok = idx[p] >= 0
            want[p].index_add_(0, idx[p][ok], g.reshape(rows, num_pq, d)[ok, p])
        assert torch.equal(native.code_lookup_grad(g.to(dev), idx.to(dev), k).cpu(), want), kind
